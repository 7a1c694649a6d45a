// C ABI of the products of rows grouped by expert (include/cumpsgemm/cumpsgemm_ext.h): checks of the
// arguments, workspace, and what has to be done to the operands in front of the kernel.
#include "activation.cuh"
#include "block_scale.cuh"
#include "grouped.hpp"

#include <cumpsgemm/cumpsgemm_ext.h>

namespace cumpsgemm_b200 {
namespace {

constexpr uint64_t kMaxDim = 0x7fffffffull - 512; // sizes and tile numbers are 32-bit in the kernels

uint64_t round_up(uint64_t x, uint64_t a) { return (x + a - 1) / a * a; }

cublasStatus_t refuse(const char *where, const char *why) {
  log_error(std::string(where) + ": " + why);
  return CUBLAS_STATUS_INVALID_VALUE;
}

bool known_type(cudaDataType_t t) { return t == CUDA_R_16F || t == CUDA_R_16BF || t == CUDA_R_32F; }
GroupedOut out_type(cudaDataType_t t) {
  return t == CUDA_R_32F ? GroupedOut::f32 : t == CUDA_R_16BF ? GroupedOut::bf16 : GroupedOut::f16;
}

// What TMA asks of a matrix: 16-byte aligned, rows and matrices multiples of 16 bytes apart (and less
// than 2^40).
bool tma_can_read(const GroupedOperand &o, int elem_bytes) {
  const uint64_t es = static_cast<uint64_t>(elem_bytes), limit = 1ull << 40;
  return (reinterpret_cast<uintptr_t>(o.ptr) & 15u) == 0 && o.ld * es % 16 == 0 &&
         (o.batch == 1 || o.stride * es % 16 == 0) && o.ld * es < limit &&
         (o.batch == 1 || o.stride * es < limit);
}

// Lays the operands out for the kernel where they are not so already: FP32 is split, rows that TMA
// cannot address are copied.  elem_bytes: of the source.  On success the operands point to what the
// kernel reads.
cublasStatus_t stage(cuMpSGEMM_handle *h, const char *where, GroupedArgs &g, int elem_bytes,
                     bool a_is_weights, bool scale) {
  StageArgs s = {};
  s.elem_bytes = elem_bytes;
  s.ends = g.ends;
  s.rows = g.rows;
  s.groups = g.groups;
  s.scale = scale;
  const uint64_t dst_elem = elem_bytes == 1 ? 1 : 2, per16 = 16 / dst_elem;
  uint64_t bytes = 0, offset[2] = {0, 0};
  GroupedOperand *op[2] = {&g.a, &g.b}, *moved[2];
  for (int i = 0; i < 2; ++i) {
    GroupedOperand &o = *op[i];
    if (o.outer == 0) { // no rows: nothing is read, but the kernel's map wants a whole row
      o.ld = round_up(o.inner, per16);
      o.planes = elem_bytes == 4 ? 2 : 1;
      o.plane_stride = o.ld;
      continue;
    }
    if (elem_bytes != 4 && tma_can_read(o, elem_bytes)) continue;
    StageOperand &d = s.op[s.count];
    d.src = o.ptr;
    d.ld = o.ld;
    d.stride = o.stride;
    d.inner = o.inner;
    d.outer = o.outer;
    d.batch = o.batch;
    d.ld_dst = round_up(o.inner, per16);
    d.rows_are_grouped = !(i == 0 && a_is_weights);
    o.planes = elem_bytes == 4 ? 2 : 1;
    o.ld = d.ld_dst;
    o.stride = o.outer * o.ld;
    o.plane_stride = o.batch * o.stride;
    offset[s.count] = bytes;
    bytes += round_up(o.planes * o.plane_stride * dst_elem, 1024);
    moved[s.count++] = &o;
  }
  const uint64_t records_at = bytes;
  if (scale && s.count > 0) bytes += round_up((2 * kScaleRecords + 2) * sizeof(float), 1024);
  const uint64_t scratch_at = bytes;
  bytes += round_up(g.scratch_bytes, 1024);
  // the sums of slices are a matter of speed: without room for them tiles stay whole
  const uint64_t parts_at = bytes, parts = grouped_parts_bytes(g, h->num_sms);
  const bool with_parts = parts > 0 && bytes + parts <= workspace_limit(h) && ensure_workspace(h, bytes + parts);
  if (!with_parts && bytes > 0 && (bytes > workspace_limit(h) || !ensure_workspace(h, bytes))) {
    if (g.scratch_bytes == 0) // (else the caller has another way)
      log_error(std::string(where) + ": no workspace of " + std::to_string(bytes >> 20) + " MB for the operands");
    return CUBLAS_STATUS_ALLOC_FAILED;
  }
  char *ws = static_cast<char *>(h->workspace);
  if (with_parts) g.parts = reinterpret_cast<float *>(ws + parts_at);
  if (g.scratch_bytes > 0) g.scratch = ws + scratch_at;
  g.counters = h->dev_grouped_counters;
  if (s.count == 0) return CUBLAS_STATUS_SUCCESS;
  for (int i = 0; i < s.count; ++i) {
    s.op[i].dst = ws + offset[i];
    moved[i]->ptr = ws + offset[i];
  }
  if (scale) {
    s.records = reinterpret_cast<float *>(ws + records_at);
    s.unscale = s.records + 2 * kScaleRecords;
    g.unscale = s.unscale;
  }
  return launch_stage(s, h->num_sms, h->cuda_stream) == cudaSuccess ? CUBLAS_STATUS_SUCCESS
                                                                    : CUBLAS_STATUS_EXECUTION_FAILED;
}

cublasStatus_t finish(cuMpSGEMM_handle *h, const GroupedArgs &g) {
  const cudaError_t e = launch_grouped_gemm(g, h->cuda_stream);
  mark_stream_work(h);
  return e == cudaSuccess ? CUBLAS_STATUS_SUCCESS : CUBLAS_STATUS_EXECUTION_FAILED;
}

// Sizes common to all products.
const char *check_sizes(uint64_t rows, uint64_t n, uint64_t k, uint32_t groups, const int32_t *ends) {
  if (n == 0 || k == 0 || groups == 0) return "n, k and the number of groups must not be 0";
  if (groups > kMaxGroups) return "more than 1024 groups";
  if (ends == nullptr && groups != 1) return "group_ends is needed for more than one group";
  if (rows > kMaxDim || n > kMaxDim || k > kMaxDim) return "a size does not fit 31 bits";
  // tiles of 256 x 256: of rows by n (product), or of n by k for every group (gradient of the weights)
  if ((rows / 256 + groups + 2) * (n / 256 + 1) > kMaxDim ||
      groups * (n / 256 + 1) * (k / 256 + 1) > kMaxDim)
    return "too many tiles";
  return nullptr;
}

// Whether an FP32 product goes to the kernel for few rows, which passes over a group's weights once for
// every 8 of its rows: up to 6 for each group on average.  How they are spread is known on the device only.  Evenly
// it is the shorter way, by half and more: 16 groups of 2048 x 4096 with 6 rows each 185 us against 263, 64 of
// 2048 x 2048 285 against 508.  With all of those rows in one group there is less to read for both: 97 against
// 41 and 143 (stored n by k 190) against 52, so the most it costs is less than what it saves.
bool takes_few_rows(uint64_t rows, uint32_t groups) { return rows <= 6ull * groups; }

bool known_activation(int a) { return a >= 0 && a <= static_cast<int>(Activation::relu); }
bool known_f8(cudaDataType_t t) { return t == CUDA_R_8F_E4M3 || t == CUDA_R_8F_E5M2; }
int f8_type(cudaDataType_t t) { return static_cast<int>(t == CUDA_R_8F_E4M3 ? F8Type::e4m3 : F8Type::e5m2); }
cublasStatus_t done(cuMpSGEMM_handle *h, cudaError_t e) {
  mark_stream_work(h);
  return e == cudaSuccess ? CUBLAS_STATUS_SUCCESS : CUBLAS_STATUS_EXECUTION_FAILED;
}

// Whether a gated product of 16-bit operands goes to the kernel that passes over a group's weights once for every 8 of its
// rows: a call of 8 rows or fewer, which so meets no weights twice.  One row or 8 of 4096 x 2 x 4096 14 us against 18,
// of 1024 x 2 x 1024 2.9 against 9.4, 8 rows over as many experts of 512 x 2 x 512 4.4 against 8.7; no difference where
// memory alone counts (8192 x 2 x 8192 49 and 48).  With more rows the other one is the faster: 64 over as many experts of 2048 x 2 x
// 2048 160 us against 174, all 64 of one expert 13 against 42.
bool gated_takes_few_rows(const GroupedArgs &g) {
  return g.rows <= 8 && g.k % 8 == 0 && tma_can_read(g.a, 2) && tma_can_read(g.b, 2);
}

// Whether a product of 8-bit floating-point operands goes to the kernel for groups of few rows, which passes over a
// group's weights once for every 64 of its rows, and whose tiles are half as high and half as wide.  Up to 32 rows for
// each group on average, however they are spread: 32 groups of 4096 x 4096 with 32 rows each 85 us against 125; with all
// of those rows in one group some 50 against 30.  One group with up to 64 rows, and any call whose tiles all have an SM of
// their own: 256 rows of 4096 x 4096 15 against 21 (512, which are more tiles than that, 25 against 19).  What it costs where
// all rows are in one group grows with them, and so does what it saves where they are not: 128 groups of 4096 x 4096
// with 4096 rows 173 us against 79, evenly spread 332 against 519; 256 of 4096 x 2048 with 8192 rows 183 against 78, and 343 against 568.
bool f8_takes_few_rows(uint64_t rows, uint64_t n, uint32_t groups, unsigned num_sms) {
  const uint64_t most_tiles = (rows + 63ull * groups) / 64 * ((n + 127) / 128);
  return rows <= (groups == 1 ? 64ull : 32ull * groups) || most_tiles <= num_sms;
}

bool fp32_mode_ok(cuMpSGEMM_compute_mode_t mode) {
  return mode == CUMPSGEMM_FP16TCEC || mode == CUMPSGEMM_FP16TCEC_SCALING;
}

} // namespace
} // namespace cumpsgemm_b200

using namespace cumpsgemm_b200;

extern "C" cublasStatus_t cuMpSGEMM_grouped_gemm(
    cuMpSGEMM_handle_t h, cublasOperation_t op_W, uint64_t rows, uint64_t n, uint64_t k,
    uint32_t num_groups, const int32_t *group_ends, const float *alpha, const void *x, uint64_t ldx,
    const void *w, uint64_t ldw, uint64_t stridew, const float *beta, void *y, uint64_t ldy,
    cudaDataType_t type, cuMpSGEMM_compute_mode_t mode) {
  static const char where[] = "cuMpSGEMM_grouped_gemm";
  if (h == nullptr) return CUBLAS_STATUS_NOT_INITIALIZED;
  if (const char *why = check_sizes(rows, n, k, num_groups, group_ends)) return refuse(where, why);
  if (!known_type(type)) return refuse(where, "type is not CUDA_R_16F, CUDA_R_16BF or CUDA_R_32F");
  if (op_W != CUBLAS_OP_N && op_W != CUBLAS_OP_T && op_W != CUBLAS_OP_C)
    return refuse(where, "unknown op_W");
  if (alpha == nullptr || beta == nullptr || w == nullptr ||
      (rows > 0 && (x == nullptr || y == nullptr)))
    return refuse(where, "null pointer");
  const bool w_n_contig = op_W == CUBLAS_OP_N; // stored k by n, else n by k
  const uint64_t w_inner = w_n_contig ? n : k, w_outer = w_n_contig ? k : n;
  if (ldx < k || ldy < n || ldw < w_inner ||
      (num_groups > 1 && stridew < (w_outer - 1) * ldw + w_inner))
    return refuse(where, "a leading dimension or the stride of w is too small");
  if (type == CUDA_R_32F && !fp32_mode_ok(mode)) {
    log_error(std::string(where) + ": FP32 operands take FP16TCEC or FP16TCEC_SCALING");
    return CUBLAS_STATUS_NOT_SUPPORTED;
  }
  if (rows == 0) return CUBLAS_STATUS_SUCCESS;

  DeviceGuard guard(h->device);
  if (type == CUDA_R_32F && takes_few_rows(rows, num_groups)) {
    const FewRowsArgs f = {w_n_contig, group_ends, static_cast<const float *>(x), static_cast<const float *>(w),
                           static_cast<float *>(y), ldx, ldw, stridew, ldy, static_cast<uint32_t>(rows),
                           num_groups, static_cast<uint32_t>(n), static_cast<uint32_t>(k), *alpha, *beta};
    const cudaError_t e = launch_few_rows(f, h->num_sms, h->cuda_stream);
    mark_stream_work(h);
    return e == cudaSuccess ? CUBLAS_STATUS_SUCCESS : CUBLAS_STATUS_EXECUTION_FAILED;
  }
  GroupedArgs g = {};
  g.kind = type == CUDA_R_32F ? GroupedKind::tcec : GroupedKind::f16;
  g.out_type = out_type(type);
  g.bf16 = type == CUDA_R_16BF;
  g.a_lane_contig = w_n_contig;
  g.a = {w, w_inner, w_outer, ldw, stridew, 0, num_groups, 1};
  g.b = {x, k, rows, ldx, 0, 0, 1, 1};
  g.ends = group_ends;
  g.rows = static_cast<uint32_t>(rows);
  g.groups = num_groups;
  g.lane_dim = static_cast<uint32_t>(n);
  g.k = static_cast<uint32_t>(k);
  g.out = y;
  g.ldo = ldy;
  g.alpha = *alpha;
  g.beta = *beta;
  g.dev_status = h->dev_status;
  const cublasStatus_t st = stage(h, where, g, type == CUDA_R_32F ? 4 : 2, true,
                                  type == CUDA_R_32F && mode == CUMPSGEMM_FP16TCEC_SCALING);
  return st == CUBLAS_STATUS_SUCCESS ? finish(h, g) : st;
}

extern "C" cublasStatus_t cuMpSGEMM_grouped_gemm_wgrad(
    cuMpSGEMM_handle_t h, cublasOperation_t op_W, uint64_t rows, uint64_t n, uint64_t k,
    uint32_t num_groups, const int32_t *group_ends, const float *alpha, const void *x, uint64_t ldx,
    const void *dy, uint64_t lddy, const float *beta, void *dw, uint64_t lddw, uint64_t stridedw,
    cudaDataType_t type, cuMpSGEMM_compute_mode_t mode) {
  static const char where[] = "cuMpSGEMM_grouped_gemm_wgrad";
  if (h == nullptr) return CUBLAS_STATUS_NOT_INITIALIZED;
  if (const char *why = check_sizes(rows, n, k, num_groups, group_ends)) return refuse(where, why);
  if (!known_type(type)) return refuse(where, "type is not CUDA_R_16F, CUDA_R_16BF or CUDA_R_32F");
  if (op_W != CUBLAS_OP_N && op_W != CUBLAS_OP_T && op_W != CUBLAS_OP_C)
    return refuse(where, "unknown op_W");
  if (alpha == nullptr || beta == nullptr || dw == nullptr ||
      (rows > 0 && (x == nullptr || dy == nullptr)))
    return refuse(where, "null pointer");
  const bool w_n_contig = op_W == CUBLAS_OP_N;
  const uint64_t w_inner = w_n_contig ? n : k, w_outer = w_n_contig ? k : n;
  if (ldx < k || lddy < n || lddw < w_inner ||
      (num_groups > 1 && stridedw < (w_outer - 1) * lddw + w_inner))
    return refuse(where, "a leading dimension or the stride of dw is too small");
  if (type == CUDA_R_32F && !fp32_mode_ok(mode)) {
    log_error(std::string(where) + ": FP32 operands take FP16TCEC or FP16TCEC_SCALING");
    return CUBLAS_STATUS_NOT_SUPPORTED;
  }

  DeviceGuard guard(h->device);
  GroupedArgs g = {};
  g.kind = type == CUDA_R_32F ? GroupedKind::tcec : GroupedKind::f16;
  g.out_type = out_type(type);
  g.wgrad = true;
  g.bf16 = type == CUDA_R_16BF;
  g.a_lane_contig = true;
  const GroupedOperand ox = {x, k, rows, ldx, 0, 0, 1, 1}, ody = {dy, n, rows, lddy, 0, 0, 1, 1};
  g.a = w_n_contig ? ody : ox; // the contiguous dimension of dw
  g.b = w_n_contig ? ox : ody;
  g.ends = group_ends;
  g.rows = static_cast<uint32_t>(rows);
  g.groups = num_groups;
  g.lane_dim = static_cast<uint32_t>(w_inner);
  g.col_dim = static_cast<uint32_t>(w_outer);
  g.out = dw;
  g.ldo = lddw;
  g.stride_o = stridedw;
  g.alpha = *alpha;
  g.beta = *beta;
  g.dev_status = h->dev_status;
  const cublasStatus_t st = stage(h, where, g, type == CUDA_R_32F ? 4 : 2, false,
                                  type == CUDA_R_32F && mode == CUMPSGEMM_FP16TCEC_SCALING);
  return st == CUBLAS_STATUS_SUCCESS ? finish(h, g) : st;
}

extern "C" cublasStatus_t cuMpSGEMM_i8_grouped_gemm(
    cuMpSGEMM_handle_t h, uint64_t rows, uint64_t n, uint64_t k, uint32_t num_groups,
    const int32_t *group_ends, const int8_t *xq, uint64_t ldx, const float *x_scale, const int8_t *wq,
    uint64_t ldw, uint64_t stridew, const float *w_scale, const float *bias, void *y, uint64_t ldy,
    cudaDataType_t y_type) {
  static const char where[] = "cuMpSGEMM_i8_grouped_gemm";
  if (h == nullptr) return CUBLAS_STATUS_NOT_INITIALIZED;
  if (const char *why = check_sizes(rows, n, k, num_groups, group_ends)) return refuse(where, why);
  if (k > kMaxK8) return refuse(where, "k above 131071: the integer sums could overflow");
  if (!known_type(y_type)) return refuse(where, "y_type is not CUDA_R_16F, CUDA_R_16BF or CUDA_R_32F");
  if (wq == nullptr || w_scale == nullptr ||
      (rows > 0 && (xq == nullptr || x_scale == nullptr || y == nullptr)))
    return refuse(where, "null pointer");
  if (ldx < k || ldy < n || ldw < k || (num_groups > 1 && stridew < (n - 1) * ldw + k))
    return refuse(where, "a leading dimension or the stride of wq is too small");
  if (rows == 0) return CUBLAS_STATUS_SUCCESS;

  DeviceGuard guard(h->device);
  GroupedArgs g = {};
  g.kind = GroupedKind::i8;
  g.out_type = out_type(y_type);
  g.a = {wq, k, n, ldw, stridew, 0, num_groups, 1};
  g.b = {xq, k, rows, ldx, 0, 0, 1, 1};
  g.ends = group_ends;
  g.rows = static_cast<uint32_t>(rows);
  g.groups = num_groups;
  g.lane_dim = static_cast<uint32_t>(n);
  g.k = static_cast<uint32_t>(k);
  g.out = y;
  g.ldo = ldy;
  g.alpha = 1.f;
  g.lane_scale = w_scale;
  g.col_scale = x_scale;
  g.bias = bias;
  g.dev_status = h->dev_status;
  const cublasStatus_t st = stage(h, where, g, 1, true, false);
  return st == CUBLAS_STATUS_SUCCESS ? finish(h, g) : st;
}

extern "C" cublasStatus_t cuMpSGEMM_quantize_rows_i8(cuMpSGEMM_handle_t h, uint64_t rows, uint64_t k,
                                                     const void *x, uint64_t ldx, cudaDataType_t type,
                                                     const int32_t *row_index, uint64_t src_rows,
                                                     int8_t *q, uint64_t ldq, float *scale) {
  static const char where[] = "cuMpSGEMM_quantize_rows_i8";
  if (h == nullptr) return CUBLAS_STATUS_NOT_INITIALIZED;
  if (k == 0) return refuse(where, "k must not be 0");
  if (rows > kMaxDim || k > kMaxDim || src_rows > kMaxDim)
    return refuse(where, "a size does not fit 31 bits");
  if (!known_type(type)) return refuse(where, "type is not CUDA_R_16F, CUDA_R_16BF or CUDA_R_32F");
  if (ldx < k || ldq < k) return refuse(where, "a leading dimension is too small");
  if (rows > 0 && (q == nullptr || scale == nullptr || (src_rows > 0 && x == nullptr)))
    return refuse(where, "null pointer");
  if (row_index == nullptr && src_rows < rows)
    return refuse(where, "fewer rows in x than asked for, and no row_index");
  if (rows == 0) return CUBLAS_STATUS_SUCCESS;

  DeviceGuard guard(h->device);
  QuantizeArgs a = {};
  a.x = x;
  a.type = static_cast<int>(out_type(type));
  a.ldx = ldx;
  a.row_index = row_index;
  a.src_rows = static_cast<uint32_t>(src_rows);
  a.rows = static_cast<uint32_t>(rows);
  a.k = static_cast<uint32_t>(k);
  a.q = q;
  a.ldq = ldq;
  a.scale = scale;
  const cudaError_t e = launch_quantize_rows(a, h->num_sms, h->cuda_stream);
  mark_stream_work(h);
  return e == cudaSuccess ? CUBLAS_STATUS_SUCCESS : CUBLAS_STATUS_EXECUTION_FAILED;
}

static cublasStatus_t gated_rows(cuMpSGEMM_handle_t h, uint64_t rows, uint64_t hidden, const void *pre, uint64_t ldpre,
                                 const void *dh, uint64_t lddh, int activation, void *out, uint64_t ldo,
                                 cudaDataType_t type) {
  GatedRowsArgs a = {};
  a.pre = pre;
  a.dh = dh;
  a.type = static_cast<int>(out_type(type));
  a.activation = activation;
  a.ldpre = ldpre;
  a.lddh = lddh;
  a.ldo = ldo;
  a.rows = static_cast<uint32_t>(rows);
  a.hidden = static_cast<uint32_t>(hidden);
  a.out = out;
  return done(h, launch_gated_rows(a, h->num_sms, h->cuda_stream));
}

extern "C" cublasStatus_t cuMpSGEMM_gated_rows(cuMpSGEMM_handle_t h, uint64_t rows, uint64_t hidden, const void *pre,
                                               uint64_t ldpre, const void *dh, uint64_t lddh,
                                               cuMpSGEMM_activation_t activation, void *out, uint64_t ldo,
                                               cudaDataType_t type) {
  static const char where[] = "cuMpSGEMM_gated_rows";
  if (h == nullptr) return CUBLAS_STATUS_NOT_INITIALIZED;
  if (hidden == 0) return refuse(where, "hidden must not be 0");
  if (rows > kMaxDim || hidden > kMaxDim / 2) return refuse(where, "a size does not fit 31 bits");
  if (!known_type(type)) return refuse(where, "type is not CUDA_R_16F, CUDA_R_16BF or CUDA_R_32F");
  if (!known_activation(activation)) return refuse(where, "unknown activation");
  if (ldpre < 2 * hidden || (dh != nullptr && lddh < hidden) || ldo < (dh != nullptr ? 2 * hidden : hidden))
    return refuse(where, "a leading dimension is too small");
  if (rows > 0 && (pre == nullptr || out == nullptr)) return refuse(where, "null pointer");
  if (rows == 0) return CUBLAS_STATUS_SUCCESS;
  DeviceGuard guard(h->device);
  return gated_rows(h, rows, hidden, pre, ldpre, dh, lddh, activation, out, ldo, type);
}

extern "C" cublasStatus_t cuMpSGEMM_grouped_gemm_gated(
    cuMpSGEMM_handle_t h, uint64_t rows, uint64_t hidden, uint64_t k, uint32_t num_groups, const int32_t *group_ends,
    const void *x, uint64_t ldx, const void *w, uint64_t ldw, uint64_t stridew, cuMpSGEMM_activation_t activation,
    void *y, uint64_t ldy, void *pre, uint64_t ldpre, cudaDataType_t type, cuMpSGEMM_compute_mode_t mode) {
  static const char where[] = "cuMpSGEMM_grouped_gemm_gated";
  if (h == nullptr) return CUBLAS_STATUS_NOT_INITIALIZED;
  if (hidden > kMaxDim / 2) return refuse(where, "a size does not fit 31 bits");
  if (const char *why = check_sizes(rows, 2 * hidden, k, num_groups, group_ends)) return refuse(where, why);
  if (!known_type(type)) return refuse(where, "type is not CUDA_R_16F, CUDA_R_16BF or CUDA_R_32F");
  if (!known_activation(activation)) return refuse(where, "unknown activation");
  if (w == nullptr || (rows > 0 && (x == nullptr || y == nullptr || (pre == nullptr && type == CUDA_R_32F))))
    return refuse(where, "null pointer");
  if (ldx < k || ldy < hidden || ldw < k || (num_groups > 1 && stridew < (2 * hidden - 1) * ldw + k) ||
      (pre != nullptr && ldpre < 2 * hidden))
    return refuse(where, "a leading dimension or the stride of w is too small");
  if (type == CUDA_R_32F && !fp32_mode_ok(mode)) {
    log_error(std::string(where) + ": FP32 operands take FP16TCEC or FP16TCEC_SCALING");
    return CUBLAS_STATUS_NOT_SUPPORTED;
  }
  if (rows == 0) return CUBLAS_STATUS_SUCCESS;

  if (type != CUDA_R_32F) {
    DeviceGuard guard(h->device);
    GroupedArgs g = {};
    g.kind = GroupedKind::f16;
    g.out_type = out_type(type);
    g.bf16 = type == CUDA_R_16BF;
    g.a = {w, k, 2 * hidden, ldw, stridew, 0, num_groups, 1};
    g.b = {x, k, rows, ldx, 0, 0, 1, 1};
    g.ends = group_ends;
    g.rows = static_cast<uint32_t>(rows);
    g.groups = num_groups;
    g.lane_dim = static_cast<uint32_t>(2 * hidden);
    g.k = static_cast<uint32_t>(k);
    g.out = y;
    g.ldo = ldy;
    g.alpha = 1.f;
    g.dev_status = h->dev_status;
    g.gated = GatedKind::gated;
    g.activation = activation;
    g.pre = pre;
    g.ldpre = ldpre;
    if (gated_takes_few_rows(g)) return done(h, launch_gated_few_rows(g, h->cuda_stream));
    const cublasStatus_t st = stage(h, where, g, 2, true, false);
    return st == CUBLAS_STATUS_SUCCESS ? finish(h, g) : st;
  }
  const float one = 1.f, zero = 0.f;
  const cublasStatus_t st = cuMpSGEMM_grouped_gemm(h, CUBLAS_OP_T, rows, 2 * hidden, k, num_groups, group_ends, &one, x, ldx,
                                                   w, ldw, stridew, &zero, pre, ldpre, type, mode);
  if (st != CUBLAS_STATUS_SUCCESS) return st;
  DeviceGuard guard(h->device);
  return gated_rows(h, rows, hidden, pre, ldpre, nullptr, 0, activation, y, ldy, type);
}

extern "C" cublasStatus_t cuMpSGEMM_grouped_gemm_gated_grad(
    cuMpSGEMM_handle_t h, cublasOperation_t op_W, uint64_t rows, uint64_t hidden, uint64_t k, uint32_t num_groups,
    const int32_t *group_ends, const void *dy, uint64_t lddy, const void *w, uint64_t ldw, uint64_t stridew,
    cuMpSGEMM_activation_t activation, const void *pre, uint64_t ldpre, void *dpre, uint64_t lddpre,
    cudaDataType_t type, cuMpSGEMM_compute_mode_t mode) {
  static const char where[] = "cuMpSGEMM_grouped_gemm_gated_grad";
  if (h == nullptr) return CUBLAS_STATUS_NOT_INITIALIZED;
  if (hidden > kMaxDim / 2) return refuse(where, "a size does not fit 31 bits");
  if (const char *why = check_sizes(rows, hidden, k, num_groups, group_ends)) return refuse(where, why);
  if (!known_type(type)) return refuse(where, "type is not CUDA_R_16F, CUDA_R_16BF or CUDA_R_32F");
  if (!known_activation(activation)) return refuse(where, "unknown activation");
  if (op_W != CUBLAS_OP_N && op_W != CUBLAS_OP_T && op_W != CUBLAS_OP_C) return refuse(where, "unknown op_W");
  if (w == nullptr || (rows > 0 && (dy == nullptr || pre == nullptr || dpre == nullptr))) return refuse(where, "null pointer");
  const bool w_n_contig = op_W == CUBLAS_OP_N;
  const uint64_t w_inner = w_n_contig ? hidden : k, w_outer = w_n_contig ? k : hidden;
  if (lddy < k || ldpre < 2 * hidden || lddpre < 2 * hidden || ldw < w_inner ||
      (num_groups > 1 && stridew < (w_outer - 1) * ldw + w_inner))
    return refuse(where, "a leading dimension or the stride of w is too small");
  if (type == CUDA_R_32F && !fp32_mode_ok(mode)) {
    log_error(std::string(where) + ": FP32 operands take FP16TCEC or FP16TCEC_SCALING");
    return CUBLAS_STATUS_NOT_SUPPORTED;
  }
  if (rows == 0) return CUBLAS_STATUS_SUCCESS;

  if (type != CUDA_R_32F) {
    DeviceGuard guard(h->device);
    GroupedArgs g = {};
    g.kind = GroupedKind::f16;
    g.out_type = out_type(type);
    g.bf16 = type == CUDA_R_16BF;
    g.a_lane_contig = w_n_contig;
    g.a = {w, w_inner, w_outer, ldw, stridew, 0, num_groups, 1};
    g.b = {dy, k, rows, lddy, 0, 0, 1, 1};
    g.ends = group_ends;
    g.rows = static_cast<uint32_t>(rows);
    g.groups = num_groups;
    g.lane_dim = static_cast<uint32_t>(hidden);
    g.k = static_cast<uint32_t>(k);
    g.out = dpre;
    g.ldo = lddpre;
    g.alpha = 1.f;
    g.dev_status = h->dev_status;
    g.gated = GatedKind::grad;
    g.activation = activation;
    g.pre = const_cast<void *>(pre);
    g.ldpre = ldpre;
    const cublasStatus_t st = stage(h, where, g, 2, true, false);
    return st == CUBLAS_STATUS_SUCCESS ? finish(h, g) : st;
  }
  // dh goes to the first half of dpre, and the elementwise pass takes it from there
  const float one = 1.f, zero = 0.f;
  const cublasStatus_t st = cuMpSGEMM_grouped_gemm(h, op_W, rows, hidden, k, num_groups, group_ends, &one, dy, lddy, w, ldw,
                                                   stridew, &zero, dpre, lddpre, type, mode);
  if (st != CUBLAS_STATUS_SUCCESS) return st;
  DeviceGuard guard(h->device);
  return gated_rows(h, rows, hidden, pre, ldpre, dpre, lddpre, activation, dpre, lddpre, type);
}

extern "C" cublasStatus_t cuMpSGEMM_quantize_rows_f8(cuMpSGEMM_handle_t h, uint64_t rows, uint64_t k, const void *x,
                                                     uint64_t ldx, cudaDataType_t type, const int32_t *row_index,
                                                     uint64_t src_rows, int activation, void *q, uint64_t ldq,
                                                     cudaDataType_t q_type, float *scale, uint64_t scale_row,
                                                     uint64_t scale_block) {
  static const char where[] = "cuMpSGEMM_quantize_rows_f8";
  if (h == nullptr) return CUBLAS_STATUS_NOT_INITIALIZED;
  if (k == 0) return refuse(where, "k must not be 0");
  if (rows > kMaxDim || k > kMaxDim / 2 || src_rows > kMaxDim) return refuse(where, "a size does not fit 31 bits");
  if (!known_type(type)) return refuse(where, "type is not CUDA_R_16F, CUDA_R_16BF or CUDA_R_32F");
  if (!known_f8(q_type)) return refuse(where, "q_type is not CUDA_R_8F_E4M3 or CUDA_R_8F_E5M2");
  if (activation != CUMPSGEMM_ACTIVATION_NONE && !known_activation(activation)) return refuse(where, "unknown activation");
  if (ldx < (activation == CUMPSGEMM_ACTIVATION_NONE ? k : 2 * k) || ldq < k)
    return refuse(where, "a leading dimension is too small");
  if (rows > 0 && (q == nullptr || scale == nullptr || (src_rows > 0 && x == nullptr))) return refuse(where, "null pointer");
  if (row_index == nullptr && src_rows < rows) return refuse(where, "fewer rows in x than asked for, and no row_index");
  if (rows == 0) return CUBLAS_STATUS_SUCCESS;

  DeviceGuard guard(h->device);
  BlockRowsArgs a = {};
  a.x = x;
  a.type = static_cast<int>(out_type(type));
  a.q_type = f8_type(q_type);
  a.activation = activation;
  a.ldx = ldx;
  a.row_index = row_index;
  a.src_rows = static_cast<uint32_t>(src_rows);
  a.rows = static_cast<uint32_t>(rows);
  a.k = static_cast<uint32_t>(k);
  a.q = static_cast<uint8_t *>(q);
  a.ldq = ldq;
  a.scale = scale;
  a.scale_row = scale_row;
  a.scale_block = scale_block;
  return done(h, launch_block_rows(a, h->num_sms, h->cuda_stream));
}

extern "C" cublasStatus_t cuMpSGEMM_quantize_blocks_f8(cuMpSGEMM_handle_t h, uint32_t matrices, uint64_t n, uint64_t k,
                                                       const void *w, uint64_t ldw, uint64_t stridew, cudaDataType_t type,
                                                       void *q, uint64_t ldq, uint64_t strideq, cudaDataType_t q_type,
                                                       float *scale) {
  static const char where[] = "cuMpSGEMM_quantize_blocks_f8";
  if (h == nullptr) return CUBLAS_STATUS_NOT_INITIALIZED;
  if (n == 0 || k == 0) return refuse(where, "n and k must not be 0");
  if (n > kMaxDim || k > kMaxDim) return refuse(where, "a size does not fit 31 bits");
  if (!known_type(type)) return refuse(where, "type is not CUDA_R_16F, CUDA_R_16BF or CUDA_R_32F");
  if (!known_f8(q_type)) return refuse(where, "q_type is not CUDA_R_8F_E4M3 or CUDA_R_8F_E5M2");
  if (ldw < k || ldq < k || (matrices > 1 && (stridew < (n - 1) * ldw + k || strideq < (n - 1) * ldq + k)))
    return refuse(where, "a leading dimension or stride is too small");
  if (matrices > 0 && (w == nullptr || q == nullptr || scale == nullptr)) return refuse(where, "null pointer");
  if (matrices == 0) return CUBLAS_STATUS_SUCCESS;

  DeviceGuard guard(h->device);
  WeightBlocksArgs a = {};
  a.w = w;
  a.type = static_cast<int>(out_type(type));
  a.q_type = f8_type(q_type);
  a.ldw = ldw;
  a.stridew = stridew;
  a.matrices = matrices;
  a.n = static_cast<uint32_t>(n);
  a.k = static_cast<uint32_t>(k);
  a.q = static_cast<uint8_t *>(q);
  a.ldq = ldq;
  a.strideq = strideq;
  a.scale = scale;
  return done(h, launch_weight_blocks(a, h->num_sms, h->cuda_stream));
}

// What both products of 8-bit floating-point operands check and set; n: rows of w.
static cublasStatus_t f8_product(cuMpSGEMM_handle_t h, const char *where, uint64_t rows, uint64_t n, uint64_t k,
                                 uint32_t num_groups, const int32_t *group_ends, const void *xq, uint64_t ldx,
                                 cudaDataType_t x_type, const float *x_scale, const void *wq, uint64_t ldw, uint64_t stridew,
                                 cudaDataType_t w_type, const float *w_scale, GroupedArgs &g, F8Args &f) {
  if (const char *why = check_sizes(rows, n, k, num_groups, group_ends)) return refuse(where, why);
  if (!known_f8(x_type) || !known_f8(w_type))
    return refuse(where, "x_type or w_type is not CUDA_R_8F_E4M3 or CUDA_R_8F_E5M2");
  if (wq == nullptr || w_scale == nullptr || (rows > 0 && (xq == nullptr || x_scale == nullptr || g.out == nullptr)))
    return refuse(where, "null pointer");
  if (ldx < k || ldw < k || (num_groups > 1 && stridew < (n - 1) * ldw + k))
    return refuse(where, "a leading dimension or the stride of wq is too small");
  if (rows == 0) return CUBLAS_STATUS_SUCCESS;

  DeviceGuard guard(h->device);
  f.few_rows = !f.gated && f8_takes_few_rows(rows, n, num_groups, h->num_sms);
  g.kind = GroupedKind::f8;
  g.a = {wq, k, n, ldw, stridew, 0, num_groups, 1};
  g.b = {xq, k, rows, ldx, 0, 0, 1, 1};
  g.ends = group_ends;
  g.rows = static_cast<uint32_t>(rows);
  g.groups = num_groups;
  g.k = static_cast<uint32_t>(k);
  g.lane_scale = w_scale;
  g.col_scale = x_scale;
  g.dev_status = h->dev_status;
  g.f8 = &f;
  f.x_type = f8_type(x_type);
  f.w_type = f8_type(w_type);
  const cublasStatus_t st = stage(h, where, g, 1, true, false);
  if (st != CUBLAS_STATUS_SUCCESS) return st;
  if (g.scratch_bytes > 0) g.out = g.scratch;
  return finish(h, g);
}

extern "C" cublasStatus_t cuMpSGEMM_f8_grouped_gemm(
    cuMpSGEMM_handle_t h, uint64_t rows, uint64_t n, uint64_t k, uint32_t num_groups, const int32_t *group_ends,
    const void *xq, uint64_t ldx, cudaDataType_t x_type, const float *x_scale, uint64_t x_scale_row, uint64_t x_scale_block,
    const void *wq, uint64_t ldw, uint64_t stridew, cudaDataType_t w_type, const float *w_scale, const float *bias, void *y,
    uint64_t ldy, cudaDataType_t y_type) {
  static const char where[] = "cuMpSGEMM_f8_grouped_gemm";
  if (h == nullptr) return CUBLAS_STATUS_NOT_INITIALIZED;
  if (!known_type(y_type)) return refuse(where, "y_type is not CUDA_R_16F, CUDA_R_16BF or CUDA_R_32F");
  if (ldy < n) return refuse(where, "the leading dimension of y is too small");
  GroupedArgs g = {};
  F8Args f = {};
  g.out_type = out_type(y_type);
  g.lane_dim = static_cast<uint32_t>(n);
  g.out = y;
  g.ldo = ldy;
  g.bias = bias;
  f.x_scale_row = x_scale_row;
  f.x_scale_block = x_scale_block;
  return f8_product(h, where, rows, n, k, num_groups, group_ends, xq, ldx, x_type, x_scale, wq, ldw, stridew, w_type, w_scale,
                    g, f);
}

extern "C" cublasStatus_t cuMpSGEMM_f8_grouped_gemm_gated(
    cuMpSGEMM_handle_t h, uint64_t rows, uint64_t hidden, uint64_t k, uint32_t num_groups, const int32_t *group_ends,
    const void *xq, uint64_t ldx, cudaDataType_t x_type, const float *x_scale, uint64_t x_scale_row, uint64_t x_scale_block,
    const void *wq, uint64_t ldw, uint64_t stridew, cudaDataType_t w_type, const float *w_scale,
    cuMpSGEMM_activation_t activation, void *q, uint64_t ldq, cudaDataType_t q_type, float *scale, uint64_t scale_row,
    uint64_t scale_block) {
  static const char where[] = "cuMpSGEMM_f8_grouped_gemm_gated";
  if (h == nullptr) return CUBLAS_STATUS_NOT_INITIALIZED;
  if (hidden == 0 || hidden % 128 != 0) return refuse(where, "hidden is not a multiple of 128");
  if (hidden > kMaxDim / 2) return refuse(where, "a size does not fit 31 bits");
  if (!known_activation(activation)) return refuse(where, "unknown activation");
  if (!known_f8(q_type)) return refuse(where, "q_type is not CUDA_R_8F_E4M3 or CUDA_R_8F_E5M2");
  if (ldq < hidden) return refuse(where, "the leading dimension of q is too small");
  if (rows > 0 && scale == nullptr) return refuse(where, "null pointer");
  // Few rows: the product in FP32 to the workspace, and a pass over it (256 rows over 32 groups, 4096 x 2 x 2048: 89 us
  // against 142 of the one kernel, whose way round costs a stage of weights more than memory does).
  if (rows > 0 && rows <= kMaxDim && num_groups > 0 && f8_takes_few_rows(rows, 2 * hidden, num_groups, h->num_sms) &&
      rows * 2 * hidden * sizeof(float) <= workspace_limit(h)) {
    GroupedArgs g = {};
    F8Args f = {};
    g.out_type = GroupedOut::f32;
    g.lane_dim = static_cast<uint32_t>(2 * hidden);
    g.out = q; // (checked; the workspace takes its place)
    g.ldo = 2 * hidden;
    g.scratch_bytes = rows * 2 * hidden * sizeof(float);
    f.x_scale_row = x_scale_row;
    f.x_scale_block = x_scale_block;
    const cublasStatus_t st = f8_product(h, where, rows, 2 * hidden, k, num_groups, group_ends, xq, ldx, x_type, x_scale, wq, ldw,
                                         stridew, w_type, w_scale, g, f);
    if (st == CUBLAS_STATUS_SUCCESS) {
      DeviceGuard guard(h->device);
      BlockRowsArgs a = {};
      a.x = g.scratch;
      a.type = static_cast<int>(GroupedOut::f32);
      a.q_type = f8_type(q_type);
      a.activation = activation;
      a.ldx = 2 * hidden;
      a.src_rows = a.rows = static_cast<uint32_t>(rows);
      a.k = static_cast<uint32_t>(hidden);
      a.q = static_cast<uint8_t *>(q);
      a.ldq = ldq;
      a.scale = scale;
      a.scale_row = scale_row;
      a.scale_block = scale_block;
      return done(h, launch_block_rows(a, h->num_sms, h->cuda_stream));
    }
    if (st != CUBLAS_STATUS_ALLOC_FAILED) return st; // (without room for that, the one kernel)
  }
  GroupedArgs g = {};
  F8Args f = {};
  g.lane_dim = static_cast<uint32_t>(hidden);
  g.out = q;
  g.ldo = ldq;
  f.x_scale_row = x_scale_row;
  f.x_scale_block = x_scale_block;
  f.gated = true;
  f.activation = activation;
  f.out_type = f8_type(q_type);
  f.out_scale = scale;
  f.out_scale_row = scale_row;
  f.out_scale_block = scale_block;
  return f8_product(h, where, rows, 2 * hidden, k, num_groups, group_ends, xq, ldx, x_type, x_scale, wq, ldw, stridew, w_type,
                    w_scale, g, f);
}
