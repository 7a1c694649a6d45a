// h = act(gate) * up of 16-bit operands for a handful of rows, in one launch without tensor memory.
//
//   g = sum_k x[r, k] w_e[f, k],  u = sum_k x[r, k] w_e[hidden + f, k],  h[r, f] = act(g) u     (pre = [g, u])
//
// Reading the weights of the groups with rows is all there is to do.  A block has 8 features: its warps share k, 64
// values at a time, multiply 8 rows of the gate and the same 8 of what it gates by up to 8 rows of x, a chunk of a group,
// (warp-wide products of 16 x 8 x 16), and add their sums in shared memory in the order of the warps.  A lane's fragments are 16 bytes
// of each of its rows as they lie in memory: the order of k within 32 is another one, on both sides the same.  The
// kernel for many rows (grouped_gemm.cu) has that many more steps in front of its first product and behind its last
// (tensor memory, barriers of pairs, slices to join), and tiles of 128 features of the result, which a call with few groups
// deals to its pairs unevenly.  One row of 4096 x 2 x 4096 takes 14.4 us, 4.7 TB/s, of which 2 are the launch's, and eight take
// as long.  Bound by memory: with as many FP32 multiply-adds instead of products eight rows took 40 us, and with the
// weights of one block of k on their way, or four, 16.4 and 15.
#include "activation.cuh"
#include "grouped_totals.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>

namespace cumpsgemm_b200 {
namespace {

constexpr int kThreads = kTotalsThreads;
constexpr uint32_t kWarps = kThreads / 32;
constexpr uint32_t kMostRows = 8; // of a group at a time
constexpr uint32_t kFeatures = 8; // of a block
constexpr uint32_t kBlock = 64;   // values of k that a warp takes at a time
constexpr uint32_t kAhead = 2;    // of those, whose weights are on their way together

struct GatedFewParams {
  const int32_t *ends;
  const void *x, *w;
  void *out, *pre; // pre: nullable
  uint64_t ldx, ldw, stridew, ldo, ldpre;
  uint32_t rows, groups, hidden, k;
  int activation;
};

template <class T> __device__ __forceinline__ T rounded(float v) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>) return __float2bfloat16_rn(v);
  else return __float2half_rn(v);
}
// weights, which pass once, and leave L1 to x; 0 behind the end
__device__ __forceinline__ uint4 load_once(const void *p, bool there) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (there)
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
// d += a b: a 16 x 16, rows lane / 4 and lane / 4 + 8; b 16 x 8, column lane / 4; d rows as a, columns 2 (lane % 4) on
template <class T>
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <class T> __global__ void __launch_bounds__(kThreads, 4) gated_few_rows_kernel(const GatedFewParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ float sums[kWarps][4][32];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, f0 = blockIdx.x * kFeatures;
  const uint32_t f = f0 + threadIdx.x % kFeatures, r = threadIdx.x / kFeatures; // what a thread writes (r < kMostRows)
  uint32_t all = ~0u;
  for (uint32_t number = blockIdx.y; number < all; number += gridDim.y) {
    const Chunk c = find_chunk<kMostRows>(p.ends, p.groups, p.rows, number, all);
    if (c.rows == 0) return;
    float g = 0.f, u = 0.f; // of the thread's feature and row; rows of no group: 0
    if (c.group < p.groups) {
      // features and rows behind the last are the last again, and not written
      const uint64_t mine = min(f0 + (lane >> 2), p.hidden - 1);
      const uint32_t from = 8 * (lane & 3u);
      const T *gate = static_cast<const T *>(p.w) + c.group * p.stridew + mine * p.ldw, *up = gate + p.hidden * p.ldw;
      const T *x = static_cast<const T *>(p.x) + (c.row0 + min(lane >> 2, c.rows - 1)) * p.ldx;
      float d[4] = {0.f, 0.f, 0.f, 0.f};
      for (uint32_t k0 = warp * kBlock; k0 < p.k; k0 += kAhead * kWarps * kBlock) { // (the same for all lanes)
        uint4 wg[kAhead][2], wu[kAhead][2];
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i)
#pragma unroll
          for (uint32_t j = 0; j < 2; ++j) {
            const uint32_t k = k0 + from + i * kWarps * kBlock + 32 * j;
            wg[i][j] = load_once(gate + k, k < p.k);
            wu[i][j] = load_once(up + k, k < p.k);
          }
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i)
#pragma unroll
          for (uint32_t j = 0; j < 2; ++j) {
            const uint32_t k = k0 + from + i * kWarps * kBlock + 32 * j;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (k < p.k) v = __ldg(reinterpret_cast<const uint4 *>(x + k));
            mma_16x8x16<T>(d, wg[i][j].x, wu[i][j].x, wg[i][j].y, wu[i][j].y, v.x, v.y);
            mma_16x8x16<T>(d, wg[i][j].z, wu[i][j].z, wg[i][j].w, wu[i][j].w, v.z, v.w);
          }
      }
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) sums[warp][i][lane] = d[i];
      __syncthreads();
      if (r < c.rows) {
#pragma unroll
        for (uint32_t w = 0; w < kWarps; ++w) {
          const uint32_t at = 4 * (threadIdx.x % kFeatures) + r / 2;
          g += sums[w][r & 1u][at];
          u += sums[w][2 + (r & 1u)][at];
        }
      }
    }
    if (r < c.rows && f < p.hidden) {
      const uint64_t row = c.row0 + r;
      if (p.pre != nullptr) {
        T *pre = static_cast<T *>(p.pre) + row * p.ldpre + f;
        pre[0] = rounded<T>(g);
        pre[p.hidden] = rounded<T>(u);
      }
      with_activation(p.activation, [&](auto act) {
        static_cast<T *>(p.out)[row * p.ldo + f] = rounded<T>(activate<act.value, true>(g).value * u);
      });
    }
  }
}

} // namespace

cudaError_t launch_gated_few_rows(const GroupedArgs &a, cudaStream_t stream) {
  GatedFewParams p = {};
  p.ends = a.ends;
  p.x = a.b.ptr;
  p.w = a.a.ptr;
  p.out = a.out;
  p.pre = a.pre;
  p.ldx = a.b.ld;
  p.ldw = a.a.ld;
  p.stridew = a.a.stride;
  p.ldo = a.ldo;
  p.ldpre = a.ldpre;
  p.rows = a.rows;
  p.groups = a.groups;
  p.hidden = a.lane_dim / 2;
  p.k = a.k;
  p.activation = a.activation;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.hidden + kFeatures - 1) / kFeatures, p.groups + 1 < p.rows ? p.groups + 1 : p.rows);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return a.bf16 ? cudaLaunchKernelEx(&cfg, gated_few_rows_kernel<__nv_bfloat16>, p)
                : cudaLaunchKernelEx(&cfg, gated_few_rows_kernel<__half>, p);
}

} // namespace cumpsgemm_b200
