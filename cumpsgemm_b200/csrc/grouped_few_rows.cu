// y[r, :] = alpha * x[r, :] op(w_e) + beta * y[r, :] in FP32 arithmetic, for FP32 operands whose groups have
// few rows, in one launch.
//
// A step of decoding sends a handful of rows to each expert, and reading the weights is all there is to
// do.  The tensor-core kernel (grouped_gemm.cu) wants them split first: read, written and read again, and
// with FP16TCEC_SCALING read once more.  Here each is read once, at any address, and multiplied with up to 8
// rows, a chunk of a group; other chunks of it pass over its weights again, in blocks of their own at the
// same time, so that most of them come from L2.  Weights of 16 experts, 2048 x 4096, which memory delivers
// in 82 us: 1 / 4 / 6 rows for each take 121 / 149 / 185 us stored k by n and 116 / 144 / 184 stored n by k, and
// the tensor-core kernel 265, with scaling 350; one row, 4096 x 4096, 14 and 12 us against 44 and 60; 8 experts
// of 512 x 512, 4 rows each, 5.3 against 14 and 21.  What bounds it: with one row memory, with more the
// loads of x from shared memory, one for every four weights and row.  (16 rows at a time spilled: 273 and
// 589 us.)  With all rows in one group: 384 of 64 groups of 2048 x 2048 take 143 and 190 us (evenly 285 and 340),
// 1536 of 256 of 512 x 1024 76 and 111 (122 and 150); where the chunks of a group ran one after another in
// its own blocks those took 1570 and 600, 3165 and 1290.
//
// op N (weights stored k by n): lanes side by side along n, the warps of a block share k and add their sums
// in shared memory, in the order of the warps.  op T (n by k): lanes side by side along k, a warp has
// some rows of w to itself and adds its lanes by shuffles.  The rows of x are in shared memory as FP32, a
// stretch of k at a time.  Nothing is atomic: results are the same from run to run.
#include "grouped_totals.cuh"

#include <type_traits>

namespace cumpsgemm_b200 {
namespace {

constexpr int kThreads = kTotalsThreads;
constexpr int kWarps = kThreads / 32;
constexpr uint32_t kMostRows = 8;  // of a group at a time
constexpr uint32_t kHeld = 8192;   // values of x in shared memory at a time

// four values, `have` of them (the others are 0); VEC: the address allows one access
template <bool VEC> __device__ __forceinline__ void load4(const float *p, uint32_t have, float (&v)[4]) {
  if (VEC && have >= 4) {
    const float4 x = __ldg(reinterpret_cast<const float4 *>(p));
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
  } else {
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) v[i] = i < have ? __ldg(p + i) : 0.f;
  }
}

struct FewRowsParams {
  const int32_t *ends;
  const float *x, *w;
  float *y;
  uint64_t ldx, ldw, stridew, ldy;
  uint32_t rows, groups, n, k;
  float alpha, beta;
};

// The rows of one group, at most kMostRows of them, that a block multiplies.
struct Chunk {
  uint32_t group, row0, rows; // rows == 0: there is none
};
// Chunk `number` (all threads give the same), and how many there are, by all threads.
__device__ __forceinline__ Chunk find_chunk(const FewRowsParams &p, uint32_t number, uint32_t &all) {
  __shared__ uint32_t chunks[kWarps];
  __shared__ Chunk found;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const GroupTotals t(p.ends, p.groups, p.rows);
  auto chunks_of = [&](uint32_t i) { return (t.end[i] - t.begin_of(i) + kMostRows - 1) / kMostRows; };
  uint32_t mine = 0;
#pragma unroll
  for (uint32_t i = 0; i < GroupTotals::MOST; ++i) mine += chunks_of(i);
  uint32_t at = mine; // chunks in front of the thread's
#pragma unroll
  for (uint32_t d = 1; d < 32; d <<= 1) {
    const uint32_t o = __shfl_up_sync(0xffffffffu, at, d);
    if (lane >= d) at += o;
  }
  if (lane == 31) chunks[warp] = at;
  if (threadIdx.x == 0) found.rows = 0;
  at -= mine;
  __syncthreads();
  all = 0;
#pragma unroll
  for (uint32_t w = 0; w < kWarps; ++w) {
    if (w == warp) at += all;
    all += chunks[w];
  }
  if (number >= at && number < at + mine) {
#pragma unroll
    for (uint32_t i = 0; i < GroupTotals::MOST; ++i) {
      const uint32_t n = chunks_of(i);
      if (number >= at && number < at + n) {
        const uint32_t row0 = t.begin_of(i) + (number - at) * kMostRows;
        found = {t.first + i, row0, min(t.end[i] - row0, kMostRows)};
      }
      at += n;
    }
  }
  __syncthreads();
  return found;
}

// rows [row0, row0 + R) of x, those behind `have` as 0, values k0 .. k0 + kHeld / R - 1, as far as k goes
template <int R>
__device__ __forceinline__ void fetch_x(const FewRowsParams &p, float *xs, uint32_t row0, uint32_t have,
                                        uint32_t k0) {
  constexpr uint32_t STRETCH = kHeld / R;
  const uint32_t len = min(STRETCH, p.k - k0), padded = (len + 3u) & ~3u;
#pragma unroll
  for (uint32_t r = 0; r < R; ++r)
#pragma unroll 4
    for (uint32_t c = threadIdx.x; c < padded; c += kThreads)
      xs[r * STRETCH + c] = r < have && c < len ? __ldg(p.x + (row0 + r) * p.ldx + k0 + c) : 0.f;
}

// op N.  COL_LANES lanes along n, four columns each, 32 / COL_LANES along k; a block has 4 * COL_LANES columns.
template <int R, int COL_LANES, bool VEC>
__device__ __forceinline__ void rows_n(const FewRowsParams &p, float *smem, uint64_t group, uint32_t row0,
                                       uint32_t have) {
  constexpr uint32_t STRETCH = kHeld / R, K_LANES = 32 / COL_LANES, COLS = 4 * COL_LANES, AT_ONCE = kWarps * K_LANES;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const uint32_t cl = lane % COL_LANES, kl = lane / COL_LANES;
  const uint32_t col0 = blockIdx.x * COLS, col = col0 + 4 * cl;
  const uint32_t cols = col < p.n ? min(p.n - col, 4u) : 0u;
  const float *w = p.w + group * p.stridew + col;
  float acc[R][4];
#pragma unroll
  for (int r = 0; r < R; ++r) acc[r][0] = acc[r][1] = acc[r][2] = acc[r][3] = 0.f;
  for (uint32_t k0 = 0; k0 < p.k; k0 += STRETCH) {
    __syncthreads();
    fetch_x<R>(p, smem, row0, have, k0);
    __syncthreads();
    // a lane takes 4 neighbouring values of k, then the next 4 of its own
    for (uint32_t kk = 4 * (warp * K_LANES + kl); kk < STRETCH && k0 + kk < p.k; kk += 4 * AT_ONCE) {
      float v[4][4];
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i)
        load4<VEC>(w + (k0 + kk + i) * p.ldw, k0 + kk + i < p.k ? cols : 0u, v[i]);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float4 x = *reinterpret_cast<const float4 *>(smem + r * STRETCH + kk);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[r][j] = fmaf(x.w, v[3][j], fmaf(x.z, v[2][j], fmaf(x.y, v[1][j], fmaf(x.x, v[0][j], acc[r][j]))));
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (uint32_t d = COL_LANES; d < 32; d <<= 1) acc[r][j] += __shfl_xor_sync(0xffffffffu, acc[r][j], d);
      if (kl == 0) smem[(warp * R + r) * COLS + 4 * cl + j] = acc[r][j];
    }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < R * COLS; i += kThreads) {
    const uint32_t r = i / COLS, c = col0 + i % COLS;
    if (r >= have || c >= p.n) continue;
    float sum = 0.f;
#pragma unroll
    for (int q = 0; q < kWarps; ++q) sum += smem[q * R * COLS + i];
    float *at = p.y + (row0 + r) * p.ldy + c;
    sum *= p.alpha;
    *at = p.beta != 0.f ? fmaf(p.beta, *at, sum) : sum;
  }
}

// op T.  A warp has NB rows of w.
template <int R, int NB, bool VEC>
__device__ __forceinline__ void rows_t(const FewRowsParams &p, float *smem, uint64_t group, uint32_t row0,
                                       uint32_t have) {
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const uint32_t n0 = (blockIdx.x * kWarps + warp) * NB;
  constexpr uint32_t STRETCH = kHeld / R;
  const float *w = p.w + group * p.stridew + n0 * p.ldw;
  float acc[NB][R];
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int r = 0; r < R; ++r) acc[j][r] = 0.f;
  for (uint32_t k0 = 0; k0 < p.k; k0 += STRETCH) {
    __syncthreads();
    fetch_x<R>(p, smem, row0, have, k0);
    __syncthreads();
#pragma unroll 2
    for (uint32_t kk = 4 * lane; kk < STRETCH && k0 + kk < p.k; kk += 128) {
      const uint32_t k = k0 + kk, left = p.k - k;
      float v[NB][4];
#pragma unroll
      for (uint32_t j = 0; j < NB; ++j) load4<VEC>(w + j * p.ldw + k, n0 + j < p.n ? left : 0u, v[j]);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float4 x = *reinterpret_cast<const float4 *>(smem + r * STRETCH + kk);
#pragma unroll
        for (int j = 0; j < NB; ++j)
          acc[j][r] = fmaf(x.w, v[j][3], fmaf(x.z, v[j][2], fmaf(x.y, v[j][1], fmaf(x.x, v[j][0], acc[j][r]))));
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float sum = acc[j][r];
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      if (lane == static_cast<uint32_t>((j * R + r) % 32) && r < have && n0 + j < p.n) {
        float *at = p.y + (row0 + r) * p.ldy + n0 + j;
        sum *= p.alpha;
        *at = p.beta != 0.f ? fmaf(p.beta, *at, sum) : sum;
      }
    }
}

// SHAPE: COL_LANES (op N) or NB (op T)
template <bool OP_N, int SHAPE, bool VEC>
__global__ void __launch_bounds__(kThreads, 2) few_rows_kernel(const FewRowsParams p) {
  // (The kernel behind is not let in early: its blocks would crowd on the SMs that are free first, and go on
  // doing so from call to call; 32 experts of 512 x 2048 took 55 us or 480.)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  extern __shared__ float4 smem4[];
  float *smem = reinterpret_cast<float *>(smem4);
  // Chunks are dealt to the blocks of a column in turn: as many as groups are one each, unless some groups have
  // more rows than a chunk and others have rows too.
  uint32_t all = ~0u;
  for (uint32_t number = blockIdx.y; number < all; number += gridDim.y) {
    const Chunk c = find_chunk(p, number, all);
    if (c.rows == 0) return;
    if (c.group == p.groups) { // rows of no group
      constexpr uint32_t COLS = OP_N ? 4 * SHAPE : kWarps * SHAPE;
      for (uint32_t i = threadIdx.x; i < c.rows * COLS; i += kThreads) {
        const uint32_t col = blockIdx.x * COLS + i % COLS;
        if (col >= p.n) continue;
        float *at = p.y + (c.row0 + i / COLS) * p.ldy + col;
        *at = p.beta != 0.f ? p.beta * *at : 0.f;
      }
      continue;
    }
    auto go = [&](auto most) {
      constexpr int R = decltype(most)::value;
      if constexpr (OP_N) rows_n<R, SHAPE, VEC>(p, smem, c.group, c.row0, c.rows);
      else rows_t<R, SHAPE, VEC>(p, smem, c.group, c.row0, c.rows);
    };
    if (c.rows <= 2) go(std::integral_constant<int, 2>{});
    else if (c.rows <= 4) go(std::integral_constant<int, 4>{});
    else go(std::integral_constant<int, 8>{});
  }
}

template <bool OP_N, int SHAPE, bool VEC>
cudaError_t launch(const FewRowsParams &p, cudaStream_t stream) {
  constexpr uint32_t COLS = OP_N ? 4 * SHAPE : kWarps * SHAPE;
  constexpr size_t x_bytes = kHeld * sizeof(float),
                   sum_bytes = OP_N ? kWarps * kMostRows * COLS * sizeof(float) : 0,
                   smem = x_bytes > sum_bytes ? x_bytes : sum_bytes;
  const auto kernel = few_rows_kernel<OP_N, SHAPE, VEC>;
  static_assert(smem <= 48 * 1024, "needs no attribute");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.n + COLS - 1) / COLS, p.groups + 1 < p.rows ? p.groups + 1 : p.rows);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

} // namespace

cudaError_t launch_few_rows(const FewRowsArgs &a, unsigned num_sms, cudaStream_t stream) {
  const FewRowsParams p = {a.ends, a.x, a.w, a.y, a.ldx, a.ldw, a.stridew, a.ldy, a.rows, a.groups, a.n, a.k,
                           a.alpha, a.beta};
  const bool vec = reinterpret_cast<uintptr_t>(a.w) % 16 == 0 && a.ldw % 4 == 0 &&
                   (a.groups == 1 || a.stridew % 4 == 0);
  // Blocks are narrower where there are few: how many of the groups have rows is known on the device only, and
  // a narrow block of op N takes 5 to 28 % longer for the same weights, while 10 of 54 experts of 480 columns
  // made 40 wide blocks, which took 94 us and not 25.  (op T with one row of w for a warp was slower than with
  // two everywhere.)
  const uint64_t used = a.groups < a.rows ? a.groups : a.rows;
  if (a.op_n) {
    if (used * ((a.n + 127) / 128) >= 4ull * num_sms)
      return vec ? launch<true, 32, true>(p, stream) : launch<true, 32, false>(p, stream);
    return vec ? launch<true, 8, true>(p, stream) : launch<true, 8, false>(p, stream);
  }
  if (used * ((a.n + 31) / 32) >= num_sms)
    return vec ? launch<false, 4, true>(p, stream) : launch<false, 4, false>(p, stream);
  return vec ? launch<false, 2, true>(p, stream) : launch<false, 2, false>(p, stream);
}

} // namespace cumpsgemm_b200
