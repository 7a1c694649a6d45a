// Products of rows grouped by expert: what the kernels (grouped_gemm.cu, row_kernels.cu) and the
// entry points (grouped_api.cu) share.
#pragma once
#include "internal.hpp"

namespace cumpsgemm_b200 {

constexpr uint32_t kMaxGroups = 1024;
constexpr uint32_t kMaxK8 = 131071; // 2^14 * k has to stay below 2^31

enum class GroupedKind : int { f16 = 0, tcec = 1, i8 = 2 };
enum class GroupedOut : int { f16 = 0, bf16 = 1, f32 = 2 };

// One operand as the tensor core reads it: `planes` x `batch` matrices of `outer` rows of `inner`
// contiguous elements.  A plane is the operand itself, or (tcec) its hi and its lo half.
struct GroupedOperand {
  const void *ptr;
  uint64_t inner, outer;
  uint64_t ld, stride, plane_stride; // elements
  uint32_t batch, planes;
};

// D (lanes x columns) = A (lanes x reduction) * B (reduction x columns).  The lane dimension of the
// result is contiguous in memory.
//   product  lanes = n, columns = rows of a group, reduction = k; A = w, B = x
//   wgrad    lanes and columns = n and k, or k and n; reduction = rows of a group
struct GroupedArgs {
  GroupedKind kind;
  GroupedOut out_type;
  bool wgrad;
  bool bf16;          // kind f16: operands are bfloat16, else float16
  bool a_lane_contig; // A is stored with its lanes contiguous (wgrad: both operands are)
  GroupedOperand a, b;
  const int32_t *ends; // nullable: one group of all rows
  uint32_t rows, groups;
  uint32_t lane_dim, col_dim; // col_dim: wgrad only
  uint32_t k;                 // product only
  void *out;
  uint64_t ldo, stride_o; // elements; stride_o: wgrad only
  float alpha, beta;
  const float *unscale;    // tcec, nullable: two factors that take the scales of the operands off
  const float *lane_scale; // i8: [groups][lane_dim]
  const float *col_scale;  // i8: [rows]
  const float *bias;       // i8, nullable: [groups][lane_dim]
  float *parts; // nullable: grouped_parts_bytes() of workspace for the sums of slices
  unsigned *counters; // grouped_counters() words, zero between calls
  int *dev_status;
};
// Memory with which a call may cut tiles into slices of K; 0 where it will not.
std::size_t grouped_parts_bytes(const GroupedArgs &a, unsigned num_sms);
cudaError_t launch_grouped_gemm(const GroupedArgs &a, cudaStream_t stream);

// An operand brought into the form above: 8- or 16-bit elements copied to rows that TMA can address,
// or FP32 elements split into hi and lo FP16 planes, after a multiplication by a power of two.
struct StageOperand {
  const void *src;
  void *dst;
  uint64_t ld, stride;      // of src, elements
  uint64_t ld_dst;          // of dst, elements; a matrix of dst is outer * ld_dst elements
  uint64_t inner, outer;
  uint32_t batch;           // 1: outer runs over rows, of which those behind the last group are left out;
                            // a batch of weights leaves out the groups without rows
  bool rows_are_grouped;    // the first case
  // How the rows are dealt (launch_stage sets it): 2^lanes_log2 lanes take a segment of a row at a time,
  // of which there are `segments`, in so many steps.
  uint32_t lanes_log2, segments, steps;
};
struct StageArgs {
  StageOperand op[2];
  int count;
  int elem_bytes; // 1, 2 (copied) or 4 (split)
  const int32_t *ends;
  uint32_t rows, groups;
  bool scale;     // 4 bytes only: by the largest finite magnitude of each operand
  float *records; // scale: kScaleRecords floats for each operand
  float *unscale; // scale: two factors for the epilogue
};
constexpr uint32_t kScaleRecords = 592;
cudaError_t launch_stage(const StageArgs &a, unsigned num_sms, cudaStream_t stream);

// The product of FP32 operands in FP32 arithmetic, for groups of few rows (grouped_few_rows.cu).
struct FewRowsArgs {
  bool op_n; // w is stored k by n, else n by k
  const int32_t *ends;
  const float *x, *w;
  float *y;
  uint64_t ldx, ldw, stridew, ldy;
  uint32_t rows, groups, n, k;
  float alpha, beta;
};
cudaError_t launch_few_rows(const FewRowsArgs &a, unsigned num_sms, cudaStream_t stream);

struct QuantizeArgs {
  const void *x;
  int type; // GroupedOut
  uint64_t ldx;
  const int32_t *row_index; // nullable
  uint32_t src_rows, rows, k;
  int8_t *q;
  uint64_t ldq;
  float *scale;
};
cudaError_t launch_quantize_rows(const QuantizeArgs &a, unsigned num_sms, cudaStream_t stream);

} // namespace cumpsgemm_b200
