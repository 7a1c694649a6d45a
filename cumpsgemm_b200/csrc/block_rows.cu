// Rows and weights to 8-bit floating point with a scale for each block of 128 columns, or of 128 x 128
// (block_scale.cuh has the arithmetic), and the elementwise passes of a gated block:
//   rows     q, scale of x[row_index[r]], or of act(gate) * up of its two halves
//   weights  q, scale of each 128 x 128
//   gated    h = act(gate) * up;  backwards dgate = dh up act'(gate), dup = dh act(gate)
// A warp has a segment of a row, whose 16-byte accesses are all on their way before the first is looked at.
// What bounds them, in bfloat16:
//   rows     8192 x 8192 48 to 53 us, 3.8 to 4.2 TB/s: instructions, 79 % of the issue slots (the quotient is four for each
//            value, and all 16 lanes of a block work out its scale); memory is busy 40 % of the time
//   weights  8 x 8192 x 4096 174 us, 4.6 TB/s: neither, issue slots 60 %, memory 50 %; a block of threads meets once
//            between its loads and its stores
//   gated    8192 x 2 x 4096, silu, 43 us, 4.7 TB/s: the special-function unit, 78 %; backwards 61, 5.5 TB/s: the
//            same, 69 %, and memory, 70 %
#include "activation.cuh"
#include "block_scale.cuh"
#include "grouped.hpp"
#include "row_access.cuh"

namespace cumpsgemm_b200 {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr uint32_t kBlock = 128;

// the largest magnitude of 16 neighbouring lanes' values
__device__ __forceinline__ uint32_t half_warp_largest(uint32_t bits) {
#pragma unroll
  for (int d = 8; d > 0; d >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, d));
  return bits;
}
__device__ __forceinline__ uint32_t largest_bits(const float (&v)[8]) {
  uint32_t top = 0; // (ordered as the magnitudes, NaN above all)
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
  return top;
}
template <F8Type TYPE> __device__ __forceinline__ uint2 eight(const BlockScale &s, const float (&v)[8]) {
  return make_uint2(s.four<TYPE>(v[0], v[1], v[2], v[3]), s.four<TYPE>(v[4], v[5], v[6], v[7]));
}

// A warp takes SEGMENT columns of a row at a time: 16 lanes a block of 128, 8 values each.
constexpr uint32_t kAtOnce = 4, kSegment = kAtOnce * 2 * kBlock;

template <class T, bool WHOLE, bool GATED, F8Type TYPE>
__global__ void __launch_bounds__(kThreads) quantize_block_rows_kernel(const BlockRowsArgs a) {
  CUMPSGEMM_CHAINED_KERNEL_ENTRY();
  const uint32_t lane = threadIdx.x & 31u, segments = (a.k + kSegment - 1) / kSegment;
  const uint64_t tasks = static_cast<uint64_t>(a.rows) * segments, step = static_cast<uint64_t>(gridDim.x) * kWarps;
  uint64_t t = static_cast<uint64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  Eight<T, WHOLE> x[kAtOnce], up[GATED ? kAtOnce : 1];
  auto fetch = [&](uint64_t task) {
    const uint32_t r = static_cast<uint32_t>(task / segments);
    const uint32_t first = static_cast<uint32_t>(task - static_cast<uint64_t>(r) * segments) * (kSegment / 8) + lane;
    const int64_t from = a.row_index != nullptr ? __ldg(a.row_index + r) : static_cast<int64_t>(r);
    const bool real = from >= 0 && from < static_cast<int64_t>(a.src_rows);
    const T *row = static_cast<const T *>(a.x) + (real ? from : 0) * a.ldx;
    const uint64_t bytes = real ? a.k * static_cast<uint64_t>(sizeof(T)) : 0;
    Eight<T, WHOLE>::load(RowReader(row, bytes), first, 32, x);
    if constexpr (GATED) Eight<T, WHOLE>::load(RowReader(row + a.k, bytes), first, 32, up);
  };
  if (t < tasks) fetch(t);
  for (; t < tasks; t += step) {
    const uint32_t r = static_cast<uint32_t>(t / segments);
    const uint32_t first = static_cast<uint32_t>(t - static_cast<uint64_t>(r) * segments) * (kSegment / 8) + lane;
    float v[kAtOnce][8];
    uint32_t top[kAtOnce]; // the bits of each lane's largest magnitude
    if constexpr (GATED) {
      with_activation(a.activation, [&](auto act) {
#pragma unroll
        for (uint32_t j = 0; j < kAtOnce; ++j) {
          float u[8];
          x[j].values(v[j]);
          up[j].values(u);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[j][i] = activate<act.value, true>(v[j][i]).value * u[i];
          top[j] = largest_bits(v[j]);
        }
      });
    } else {
#pragma unroll
      for (uint32_t j = 0; j < kAtOnce; ++j) x[j].values(v[j]);
      if constexpr (sizeof(T) == 2) { // two values to an instruction, and two blocks
#pragma unroll
        for (uint32_t j = 0; j < kAtOnce; j += 2) {
          const uint32_t a0 = x[j].largest(0), a1 = x[j + 1].largest(0);
          uint32_t both = __vmaxu2(__byte_perm(a0, a1, 0x5410), __byte_perm(a0, a1, 0x7632));
#pragma unroll
          for (int d = 8; d > 0; d >>= 1) both = __vmaxu2(both, __shfl_xor_sync(0xffffffffu, both, d));
          top[j] = __float_as_uint(value_of<T>(both & 0xffffu));
          top[j + 1] = __float_as_uint(value_of<T>(both >> 16));
        }
      } else {
#pragma unroll
        for (uint32_t j = 0; j < kAtOnce; ++j) top[j] = largest_bits(v[j]);
      }
    }
    if (t + step < tasks) fetch(t + step); // on its way while this one's leaves
    if constexpr (GATED || sizeof(T) == 4) {
#pragma unroll
      for (uint32_t j = 0; j < kAtOnce; ++j) top[j] = half_warp_largest(top[j]);
    }
    uint8_t *dst = a.q + r * a.ldq;
#pragma unroll
    for (uint32_t j = 0; j < kAtOnce; ++j) {
      const BlockScale s(__uint_as_float(top[j]), TYPE);
      const uint32_t col = 8 * (first + 32 * j);
      if (col < a.k) {
        store_eight(reinterpret_cast<int8_t *>(dst), col, a.k, eight<TYPE>(s, v[j]));
        if ((lane & 15u) == 0) a.scale[r * a.scale_row + col / kBlock * a.scale_block] = s.scale;
      }
    }
  }
}

// A block of threads has a block of weights in its registers: a warp 16 rows, two at a time.
template <class T, bool WHOLE, F8Type TYPE>
__global__ void __launch_bounds__(kThreads) quantize_blocks_kernel(const WeightBlocksArgs a) {
  CUMPSGEMM_CHAINED_KERNEL_ENTRY();
  __shared__ uint32_t tops[2][kWarps];
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
  const uint32_t nb = (a.n + kBlock - 1) / kBlock, kb = (a.k + kBlock - 1) / kBlock;
  const uint64_t blocks = static_cast<uint64_t>(a.matrices) * nb * kb;
  uint32_t turn = 0;
  for (uint64_t b = blockIdx.x; b < blocks; b += gridDim.x, turn ^= 1u) {
    const uint64_t band = b / kb;
    const uint32_t col_block = static_cast<uint32_t>(b - band * kb);
    const uint32_t e = static_cast<uint32_t>(band / nb), row0 = static_cast<uint32_t>(band - static_cast<uint64_t>(e) * nb) * kBlock;
    const uint32_t col = col_block * kBlock + 8 * (lane & 15u);
    const T *w = static_cast<const T *>(a.w) + e * a.stridew;
    Eight<T, WHOLE> v[8][1];
    float x[8];
    uint32_t top = 0;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      const uint32_t row = row0 + warp * 16 + 2 * i + (lane >> 4);
      const bool real = row < a.n;
      Eight<T, WHOLE>::load(RowReader(w + (real ? row : 0) * a.ldw, real ? a.k * static_cast<uint64_t>(sizeof(T)) : 0),
                            col / 8, 0, v[i]);
    }
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      v[i][0].values(x);
      top = max(top, largest_bits(x));
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) tops[turn][warp] = top;
    __syncthreads(); // (the other turn's slots are free: everybody has passed this barrier since)
#pragma unroll
    for (int i = 0; i < kWarps; ++i) top = max(top, tops[turn][i]);
    const BlockScale s(__uint_as_float(top), TYPE);
    if (threadIdx.x == 0) a.scale[b] = s.scale;
    uint8_t *q = a.q + e * a.strideq;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      const uint32_t row = row0 + warp * 16 + 2 * i + (lane >> 4);
      v[i][0].values(x);
      if (row < a.n && col < a.k) store_eight(reinterpret_cast<int8_t *>(q + row * a.ldq), col, a.k, eight<TYPE>(s, x));
    }
  }
}

__device__ __forceinline__ void store_values(float *at, uint32_t n, const float (&v)[8]) {
  if (n == 8 && (reinterpret_cast<uintptr_t>(at) & 15u) == 0) {
    reinterpret_cast<float4 *>(at)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4 *>(at)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i)
      if (i < n) at[i] = v[i];
  }
}
template <class T> __device__ __forceinline__ T rounded(float v) {
  if constexpr (std::is_same_v<T, float>) return v;
  else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __float2bfloat16_rn(v);
  else return __float2half_rn(v);
}
template <class T> __device__ __forceinline__ float as_float(T v) {
  if constexpr (std::is_same_v<T, float>) return v;
  else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __bfloat162float(v);
  else return __half2float(v);
}
template <class T> __device__ __forceinline__ void store_values(T *at, uint32_t n, const float (&v)[8]) {
  T x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = rounded<T>(v[i]); // the one rounding to the result's type
  if (n == 8 && (reinterpret_cast<uintptr_t>(at) & 15u) == 0) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = *reinterpret_cast<const uint16_t *>(&x[2 * i]) |
             static_cast<uint32_t>(*reinterpret_cast<const uint16_t *>(&x[2 * i + 1])) << 16;
    *reinterpret_cast<uint4 *>(at) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i)
      if (i < n) at[i] = x[i];
  }
}

// One value of a gated product, or of its gradient (g: the first half, u: the second).
template <Activation ACT, class T, bool GRAD> __device__ __forceinline__ void gated_value(float &g, float &u, float d) {
  if constexpr (GRAD) gated_gradient<ACT, sizeof(T) == 2, std::is_same_v<T, __half>>(g, u, d, g, u);
  else g = activate<ACT, sizeof(T) == 2>(g).value * u;
}

constexpr uint32_t kGatedAtOnce = 2, kGatedSegment = kGatedAtOnce * 32 * 8;

// WHOLE: rows of whole aligned 16 bytes; a lane has eight neighbours.  Otherwise neighbouring lanes have neighbours: eight
// of a lane, whose stores cannot be 16 bytes, met 32 sectors at each (1999 rows x 1501 in FP32, the gradient: 31 us, and so 18).
template <class T, bool WHOLE, bool GRAD>
__global__ void __launch_bounds__(kThreads) gated_rows_kernel(const GatedRowsArgs a) {
  CUMPSGEMM_CHAINED_KERNEL_ENTRY();
  const uint32_t lane = threadIdx.x & 31u, segments = (a.hidden + kGatedSegment - 1) / kGatedSegment;
  const uint64_t tasks = static_cast<uint64_t>(a.rows) * segments, step = static_cast<uint64_t>(gridDim.x) * kWarps;
  for (uint64_t t = static_cast<uint64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5); t < tasks; t += step) {
    const uint32_t r = static_cast<uint32_t>(t / segments), seg = static_cast<uint32_t>(t - static_cast<uint64_t>(r) * segments);
    const T *pre = static_cast<const T *>(a.pre) + r * a.ldpre, *dh = static_cast<const T *>(a.dh) + r * a.lddh;
    T *out = static_cast<T *>(a.out) + r * a.ldo;
    if constexpr (WHOLE) {
      const uint64_t bytes = a.hidden * static_cast<uint64_t>(sizeof(T));
      const uint32_t first = seg * (kGatedSegment / 8) + lane;
      Eight<T, true> gate[kGatedAtOnce], up[kGatedAtOnce], back[kGatedAtOnce];
      Eight<T, true>::load(RowReader(pre, bytes), first, 32, gate);
      Eight<T, true>::load(RowReader(pre + a.hidden, bytes), first, 32, up);
      // (dh may be the first half of out: a thread reads its values before it writes there)
      if constexpr (GRAD) Eight<T, true>::template load<false>(RowReader(dh, bytes), first, 32, back);
      with_activation(a.activation, [&](auto kind) {
#pragma unroll
        for (uint32_t j = 0; j < kGatedAtOnce; ++j) {
          const uint32_t col = 8 * (first + 32 * j);
          if (col >= a.hidden) continue;
          const uint32_t n = min(8u, a.hidden - col);
          float g[8], u[8], d[8] = {};
          gate[j].values(g);
          up[j].values(u);
          if constexpr (GRAD) back[j].values(d);
#pragma unroll
          for (int i = 0; i < 8; ++i) gated_value<kind.value, T, GRAD>(g[i], u[i], d[i]);
          store_values(out + col, n, g);
          if constexpr (GRAD) store_values(out + a.hidden + col, n, u);
        }
      });
    } else {
      constexpr uint32_t N = kGatedSegment / 32;
      const uint32_t first = seg * kGatedSegment + lane;
      T gate[N], up[N], back[N];
#pragma unroll
      for (uint32_t j = 0; j < N; ++j) {
        const uint32_t col = first + 32 * j;
        if (col < a.hidden) {
          gate[j] = __ldg(pre + col);
          up[j] = __ldg(pre + a.hidden + col);
          if constexpr (GRAD) back[j] = dh[col];
        }
      }
      with_activation(a.activation, [&](auto kind) {
#pragma unroll
        for (uint32_t j = 0; j < N; ++j) {
          const uint32_t col = first + 32 * j;
          if (col >= a.hidden) continue;
          float g = as_float(gate[j]), u = as_float(up[j]);
          gated_value<kind.value, T, GRAD>(g, u, GRAD ? as_float(back[j]) : 0.f);
          out[col] = rounded<T>(g);
          if constexpr (GRAD) out[a.hidden + col] = rounded<T>(u);
        }
      });
    }
  }
}

unsigned grid_for(uint64_t warps, unsigned num_sms) {
  const uint64_t want = (warps + kWarps - 1) / kWarps, resident = static_cast<uint64_t>(num_sms) * 8;
  return static_cast<unsigned>(want < resident ? want : resident);
}
bool aligned(const void *p, uint64_t ld, uint64_t es) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld * es % 16 == 0;
}

template <class T, bool WHOLE, bool GATED>
cudaError_t block_rows(const BlockRowsArgs &a, unsigned grid, cudaStream_t stream) {
  return a.q_type == static_cast<int>(F8Type::e4m3)
             ? launch_chained(quantize_block_rows_kernel<T, WHOLE, GATED, F8Type::e4m3>, grid, kThreads, 0, stream, a)
             : launch_chained(quantize_block_rows_kernel<T, WHOLE, GATED, F8Type::e5m2>, grid, kThreads, 0, stream, a);
}
template <class T> cudaError_t block_rows(const BlockRowsArgs &a, unsigned num_sms, cudaStream_t stream) {
  // rows of whole aligned 16 bytes, the usual case: no code for ends
  const bool whole = aligned(a.x, a.ldx, sizeof(T)) && a.k * sizeof(T) % 16 == 0;
  const unsigned grid = grid_for(static_cast<uint64_t>(a.rows) * ((a.k + kSegment - 1) / kSegment), num_sms);
  if (a.activation < 0)
    return whole ? block_rows<T, true, false>(a, grid, stream) : block_rows<T, false, false>(a, grid, stream);
  return whole ? block_rows<T, true, true>(a, grid, stream) : block_rows<T, false, true>(a, grid, stream);
}

template <class T, bool WHOLE>
cudaError_t weight_blocks(const WeightBlocksArgs &a, unsigned grid, cudaStream_t stream) {
  return a.q_type == static_cast<int>(F8Type::e4m3)
             ? launch_chained(quantize_blocks_kernel<T, WHOLE, F8Type::e4m3>, grid, kThreads, 0, stream, a)
             : launch_chained(quantize_blocks_kernel<T, WHOLE, F8Type::e5m2>, grid, kThreads, 0, stream, a);
}
template <class T> cudaError_t weight_blocks(const WeightBlocksArgs &a, unsigned num_sms, cudaStream_t stream) {
  const bool whole = aligned(a.w, a.ldw, sizeof(T)) && (a.matrices == 1 || a.stridew * sizeof(T) % 16 == 0) &&
                     a.k * sizeof(T) % 16 == 0;
  const uint64_t blocks = static_cast<uint64_t>(a.matrices) * ((a.n + kBlock - 1) / kBlock) * ((a.k + kBlock - 1) / kBlock);
  const uint64_t resident = static_cast<uint64_t>(num_sms) * 4;
  const unsigned grid = static_cast<unsigned>(blocks < resident ? blocks : resident);
  return whole ? weight_blocks<T, true>(a, grid, stream) : weight_blocks<T, false>(a, grid, stream);
}

template <class T, bool WHOLE> cudaError_t gated_rows(const GatedRowsArgs &a, unsigned grid, cudaStream_t stream) {
  return a.dh == nullptr ? launch_chained(gated_rows_kernel<T, WHOLE, false>, grid, kThreads, 0, stream, a)
                         : launch_chained(gated_rows_kernel<T, WHOLE, true>, grid, kThreads, 0, stream, a);
}
template <class T> cudaError_t gated_rows(const GatedRowsArgs &a, unsigned num_sms, cudaStream_t stream) {
  const bool whole = aligned(a.pre, a.ldpre, sizeof(T)) && (a.dh == nullptr || aligned(a.dh, a.lddh, sizeof(T))) &&
                     a.hidden * sizeof(T) % 16 == 0;
  const unsigned grid =
      grid_for(static_cast<uint64_t>(a.rows) * ((a.hidden + kGatedSegment - 1) / kGatedSegment), num_sms);
  return whole ? gated_rows<T, true>(a, grid, stream) : gated_rows<T, false>(a, grid, stream);
}

} // namespace

cudaError_t launch_block_rows(const BlockRowsArgs &a, unsigned num_sms, cudaStream_t stream) {
  switch (static_cast<GroupedOut>(a.type)) {
  case GroupedOut::f32:
    return block_rows<float>(a, num_sms, stream);
  case GroupedOut::bf16:
    return block_rows<__nv_bfloat16>(a, num_sms, stream);
  default:
    return block_rows<__half>(a, num_sms, stream);
  }
}

cudaError_t launch_weight_blocks(const WeightBlocksArgs &a, unsigned num_sms, cudaStream_t stream) {
  switch (static_cast<GroupedOut>(a.type)) {
  case GroupedOut::f32:
    return weight_blocks<float>(a, num_sms, stream);
  case GroupedOut::bf16:
    return weight_blocks<__nv_bfloat16>(a, num_sms, stream);
  default:
    return weight_blocks<__half>(a, num_sms, stream);
  }
}

cudaError_t launch_gated_rows(const GatedRowsArgs &a, unsigned num_sms, cudaStream_t stream) {
  switch (static_cast<GroupedOut>(a.type)) {
  case GroupedOut::f32:
    return gated_rows<float>(a, num_sms, stream);
  case GroupedOut::bf16:
    return gated_rows<__nv_bfloat16>(a, num_sms, stream);
  default:
    return gated_rows<__half>(a, num_sms, stream);
  }
}

} // namespace cumpsgemm_b200
