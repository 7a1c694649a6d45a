// Passes over rows in front of the grouped products (grouped_gemm.cu): operands brought into a form
// that TMA and the tensor core read, and rows quantised to 8 bits.  All of them move bytes and
// little else; a warp takes a row at a time, in 16-byte accesses where the row's address allows.
#include "grouped.hpp"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace cumpsgemm_b200 {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

__device__ __forceinline__ bool finite(float v) {
  return (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u;
}

// Which rows of an operand are of use: rows in front of the last group's end; weights of groups with
// rows.  (A running total that falls back ends an empty group here as it does for the product.)
__device__ __forceinline__ uint32_t clamped_end(const int32_t *ends, uint32_t g, uint32_t rows) {
  return static_cast<uint32_t>(min(max(__ldg(ends + g), 0), static_cast<int32_t>(rows)));
}
__device__ __forceinline__ bool group_is_used(const StageArgs &a, uint32_t g) {
  if (a.ends == nullptr) return a.rows > 0;
  return clamped_end(a.ends, g, a.rows) > (g > 0 ? clamped_end(a.ends, g - 1, a.rows) : 0u);
}
// by all threads of the block
__device__ __forceinline__ uint32_t last_end(const StageArgs &a) {
  if (a.ends == nullptr) return a.rows;
  __shared__ uint32_t most;
  if (threadIdx.x == 0) most = 0;
  __syncthreads();
  uint32_t e = 0;
  for (uint32_t g = threadIdx.x; g < a.groups; g += kThreads) e = max(e, clamped_end(a.ends, g, a.rows));
  e = __reduce_max_sync(0xffffffffu, e);
  if ((threadIdx.x & 31) == 0) atomicMax(&most, e);
  __syncthreads();
  return most;
}

// The rows of all operands, one after the other, dealt to the warps of the grid.
struct RowCursor {
  uint64_t first[3]; // first row number of each operand, and their end
  uint32_t used_rows;
  __device__ __forceinline__ RowCursor(const StageArgs &a) {
    used_rows = last_end(a);
    first[0] = 0;
    for (int i = 0; i < 2; ++i)
      first[i + 1] = first[i] + (i >= a.count ? 0
                                 : a.op[i].rows_are_grouped
                                     ? static_cast<uint64_t>(used_rows)
                                     : static_cast<uint64_t>(a.op[i].batch) * a.op[i].outer);
  }
};

__device__ __forceinline__ bool aligned16(const void *p) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
}

// values i .. i + 7 of a row of n, those behind the end as 0
__device__ __forceinline__ void load8(const float *row, uint64_t i, uint64_t n, bool vec, float (&v)[8]) {
  if (vec && i + 8 <= n) {
    const float4 x = __ldg(reinterpret_cast<const float4 *>(row + i));
    const float4 y = __ldg(reinterpret_cast<const float4 *>(row + i + 4));
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = i + j < n ? row[i + j] : 0.f;
  }
}
__device__ __forceinline__ void load8(const __half *row, uint64_t i, uint64_t n, bool vec, float (&v)[8]) {
  if (vec && i + 8 <= n) {
    const uint4 x = __ldg(reinterpret_cast<const uint4 *>(row + i));
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[j]));
      v[2 * j] = f.x, v[2 * j + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = i + j < n ? __half2float(row[i + j]) : 0.f;
  }
}
__device__ __forceinline__ void load8(const __nv_bfloat16 *row, uint64_t i, uint64_t n, bool vec,
                                      float (&v)[8]) {
  if (vec && i + 8 <= n) {
    const uint4 x = __ldg(reinterpret_cast<const uint4 *>(row + i));
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      v[2 * j] = __uint_as_float(w[j] << 16), v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = i + j < n ? __bfloat162float(row[i + j]) : 0.f;
  }
}

// ---------------------------------------------------------------- scales of FP32 operands
// records[op * kScaleRecords + block] = largest finite magnitude that block met.  Infinities and NaN
// say nothing of the range of the others, and rows of no group may hold anything.
__global__ void __launch_bounds__(kThreads) largest_magnitude_kernel(const StageArgs a) {
  CUMPSGEMM_CHAINED_KERNEL_ENTRY();
  const RowCursor rows(a);
  const uint32_t lane = threadIdx.x & 31u;
  const uint64_t step = static_cast<uint64_t>(gridDim.x) * kWarps;
  float most[2] = {0.f, 0.f};
  for (uint64_t r = blockIdx.x * kWarps + (threadIdx.x >> 5); r < rows.first[2]; r += step) {
    const int o = r >= rows.first[1];
    const StageOperand &op = a.op[o];
    const uint64_t at = r - rows.first[o];
    const uint32_t b = static_cast<uint32_t>(at / op.outer);
    if (!op.rows_are_grouped && op.batch > 1 && !group_is_used(a, b)) continue;
    const float *src = static_cast<const float *>(op.src) + b * op.stride + (at - b * op.outer) * op.ld;
    const bool vec = aligned16(src);
    float m = 0.f;
    for (uint64_t i = 8ull * lane; i < op.inner; i += 256) {
      float v[8];
      load8(src, i, op.inner, vec, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) m = fmaxf(m, finite(v[j]) ? fabsf(v[j]) : 0.f);
    }
    most[o] = fmaxf(most[o], m);
  }
  __shared__ uint32_t found[2];
  if (threadIdx.x < 2) found[threadIdx.x] = 0;
  __syncthreads();
  for (int o = 0; o < 2; ++o) {
    const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(most[o])); // ordered as the values
    if (lane == 0) atomicMax(&found[o], m);
  }
  __syncthreads();
  if (threadIdx.x < 2)
    a.records[threadIdx.x * kScaleRecords + blockIdx.x] = __uint_as_float(found[threadIdx.x]);
}

// Exponent of the power of two that brings the largest magnitude to [2^14, 2^15), the scaling target
// of the other FP16TCEC_SCALING calls; at most 2^126, so operands below 2^-112 are brought up less.
__device__ __forceinline__ int scale_exponent(float largest) {
  if (largest == 0.f) return 0;
  int e;
  frexpf(largest, &e); // largest in [2^(e-1), 2^e)
  return min(15 - e, 126);
}
__device__ __forceinline__ float power_of_two(int e) { return ldexpf(1.f, e); }

// ---------------------------------------------------------------- operands into TMA's form
// BYTES 4: hi = RN_fp16(v), lo = RN_fp16((v - hi) * 2^11) for v = scale * x (split_math.cuh), in planes
// of outer * ld_dst elements for each matrix of the batch.  BYTES 1, 2: copied.
template <int BYTES>
__global__ void __launch_bounds__(kThreads) stage_kernel(const StageArgs a) {
  CUMPSGEMM_CHAINED_KERNEL_ENTRY();
  const RowCursor rows(a);
  const uint32_t lane = threadIdx.x & 31u;
  float scale[2] = {1.f, 1.f};
  if (BYTES == 4 && a.scale) {
    __shared__ uint32_t found[2];
    if (threadIdx.x < 2) found[threadIdx.x] = 0;
    __syncthreads();
    for (int o = 0; o < 2; ++o) {
      float m = 0.f;
      for (uint32_t i = threadIdx.x; i < kScaleRecords; i += kThreads)
        m = fmaxf(m, a.records[o * kScaleRecords + i]);
      const uint32_t w = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
      if (lane == 0) atomicMax(&found[o], w);
    }
    __syncthreads();
    const int e0 = scale_exponent(__uint_as_float(found[0])), e1 = scale_exponent(__uint_as_float(found[1]));
    scale[0] = power_of_two(e0);
    scale[1] = power_of_two(e1);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      // 2^-(e0 + e1) in two factors of about the same size, neither of which leaves the range
      const int e = -(e0 + e1), h = e / 2;
      a.unscale[0] = power_of_two(max(min(h, 126), -126));
      a.unscale[1] = power_of_two(max(min(e - h, 126), -126));
    }
  }
  const uint64_t step = static_cast<uint64_t>(gridDim.x) * kWarps;
  for (uint64_t r = blockIdx.x * kWarps + (threadIdx.x >> 5); r < rows.first[2]; r += step) {
    const int o = r >= rows.first[1];
    const StageOperand &op = a.op[o];
    const uint64_t at = r - rows.first[o];
    const uint32_t b = static_cast<uint32_t>(at / op.outer);
    if (!op.rows_are_grouped && op.batch > 1 && !group_is_used(a, b)) continue;
    const uint64_t src_at = b * op.stride + (at - b * op.outer) * op.ld;
    if constexpr (BYTES == 4) {
      const float *src = static_cast<const float *>(op.src) + src_at;
      const bool vec = aligned16(src);
      const float s = o ? scale[1] : scale[0];
      __half *hi = static_cast<__half *>(op.dst) + at * op.ld_dst;
      __half *lo = hi + static_cast<uint64_t>(op.batch) * op.outer * op.ld_dst;
      for (uint64_t i = 8ull * lane; i < op.inner; i += 256) {
        float v[8];
        load8(src, i, op.inner, vec, v);
        uint32_t h[4], l[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float v0 = v[2 * j] * s, v1 = v[2 * j + 1] * s;
          const __half2 hh = __floats2half2_rn(v0, v1);
          const float2 hf = __half22float2(hh);
          const __half2 ll = __floats2half2_rn((v0 - hf.x) * 2048.f, (v1 - hf.y) * 2048.f);
          h[j] = *reinterpret_cast<const uint32_t *>(&hh);
          l[j] = *reinterpret_cast<const uint32_t *>(&ll);
        }
        *reinterpret_cast<uint4 *>(hi + i) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4 *>(lo + i) = make_uint4(l[0], l[1], l[2], l[3]);
      }
    } else {
      // four bytes at a time out, byte by byte or element by element in: this is the way of
      // addresses that allow no more
      const uint8_t *src = static_cast<const uint8_t *>(op.src) + src_at * BYTES;
      uint8_t *dst = static_cast<uint8_t *>(op.dst) + at * op.ld_dst * BYTES;
      const uint64_t n = op.inner * BYTES;
      for (uint64_t i = 4ull * lane; i < n; i += 128) {
        uint32_t w = 0;
        if constexpr (BYTES == 2) {
          w = *reinterpret_cast<const uint16_t *>(src + i);
          if (i + 2 < n) w |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t *>(src + i + 2)) << 16;
        } else {
#pragma unroll
          for (uint32_t j = 0; j < 4; ++j)
            if (i + j < n) w |= static_cast<uint32_t>(src[i + j]) << (8 * j);
        }
        *reinterpret_cast<uint32_t *>(dst + i) = w;
      }
    }
  }
}

// ---------------------------------------------------------------- rows to 8 bits
// top = max_i |x_i|, scale = top / 127, q_i = rint(x_i * (127 / top)): |x_i| / top <= 1, so q_i stays
// within +-127, and an element is off by at most half a step of top / 127.  A row of zeros has scale
// 0.  A row with an infinity or NaN has no scale: its scale is NaN, its q_i are 0, and so every
// product with it is NaN.  Rows too small for 127 / top (below 2^-100) are multiplied by 2^100 first.
// A row whose index lies outside x reads as zeros.
__device__ __forceinline__ uint32_t pack4(float x, float y, float z, float w) {
  const int a = __float2int_rn(x), b = __float2int_rn(y), c = __float2int_rn(z), d = __float2int_rn(w);
  return (a & 0xff) | ((b & 0xff) << 8) | ((c & 0xff) << 16) | (static_cast<uint32_t>(d) << 24);
}

struct RowScale {
  float up, inverse, scale; // q = rint((x * up) * inverse)
  __device__ __forceinline__ explicit RowScale(uint32_t top_bits) {
    const float top = __uint_as_float(top_bits);
    up = 1.f;
    inverse = 0.f;
    scale = 0.f;
    if (top_bits >= 0x7f800000u) { // infinity or NaN, which lies above it
      up = 0.f;
      scale = __uint_as_float(0x7fffffffu);
    } else if (top > 0.f) {
      scale = __fdiv_rn(top, 127.f);
      if (top < 0x1p-100f) up = 0x1p100f;
      inverse = __fdiv_rn(127.f, top * up);
    }
  }
  __device__ __forceinline__ float operator()(float x) const { return x * up * inverse; }
};

// TPR threads to a row, which they keep in registers: VEC groups of 8 values each.
template <class T, int TPR, int VEC>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const QuantizeArgs a) {
  CUMPSGEMM_CHAINED_KERNEL_ENTRY();
  constexpr int kRowsPerBlock = kThreads / TPR;
  const uint32_t t = threadIdx.x % TPR;
  __shared__ uint32_t tops[2][kWarps];
  uint32_t turn = 0;
  for (uint64_t r = static_cast<uint64_t>(blockIdx.x) * kRowsPerBlock + threadIdx.x / TPR; r < a.rows;
       r += static_cast<uint64_t>(gridDim.x) * kRowsPerBlock, turn ^= 1u) {
    const int64_t from = a.row_index != nullptr ? __ldg(a.row_index + r) : static_cast<int64_t>(r);
    const bool real = from >= 0 && from < static_cast<int64_t>(a.src_rows);
    const T *src = static_cast<const T *>(a.x) + (real ? from : 0) * a.ldx;
    const bool vec = aligned16(src);
    float v[VEC][8];
    uint32_t top = 0; // bits of the largest magnitude; those of a NaN lie above all others
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      load8(src, 8ull * (t + j * TPR), real ? a.k : 0, vec, v[j]);
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[j][i]) & 0x7fffffffu);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if constexpr (TPR > 32) {
      if ((threadIdx.x & 31) == 0) tops[turn][threadIdx.x >> 5] = top;
      __syncthreads(); // (the other turn's slots are free: everybody has passed this barrier since)
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = max(top, tops[turn][w]);
    }
    const RowScale s(top);
    int8_t *dst = a.q + r * a.ldq;
    const bool vec_out = (reinterpret_cast<uintptr_t>(dst) & 7u) == 0;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const uint64_t i = 8ull * (t + j * TPR);
      if (i >= a.k) break;
      if (s.up == 0.f) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] = 0.f; // (not inf * 0)
      }
      const uint32_t lo = pack4(s(v[j][0]), s(v[j][1]), s(v[j][2]), s(v[j][3]));
      const uint32_t hi = pack4(s(v[j][4]), s(v[j][5]), s(v[j][6]), s(v[j][7]));
      if (vec_out && i + 8 <= a.k) {
        *reinterpret_cast<uint2 *>(dst + i) = make_uint2(lo, hi);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (i + e < a.k) dst[i + e] = static_cast<int8_t>((e < 4 ? lo >> (8 * e) : hi >> (8 * e - 32)) & 0xff);
      }
    }
    if (t == 0) a.scale[r] = s.scale;
  }
}

// Rows that no block can hold: read twice.
template <class T>
__global__ void __launch_bounds__(kThreads) quantize_long_rows_kernel(const QuantizeArgs a) {
  CUMPSGEMM_CHAINED_KERNEL_ENTRY();
  __shared__ uint32_t tops[2][kWarps];
  uint32_t turn = 0;
  for (uint64_t r = blockIdx.x; r < a.rows; r += gridDim.x, turn ^= 1u) {
    const int64_t from = a.row_index != nullptr ? __ldg(a.row_index + r) : static_cast<int64_t>(r);
    const bool real = from >= 0 && from < static_cast<int64_t>(a.src_rows);
    const T *src = static_cast<const T *>(a.x) + (real ? from : 0) * a.ldx;
    const bool vec = aligned16(src);
    const uint64_t n = real ? a.k : 0;
    uint32_t top = 0;
    for (uint64_t i = 8ull * threadIdx.x; i < n; i += 8ull * kThreads) {
      float v[8];
      load8(src, i, n, vec, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) tops[turn][threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = max(top, tops[turn][w]);
    const RowScale s(top);
    int8_t *dst = a.q + r * a.ldq;
    const bool vec_out = (reinterpret_cast<uintptr_t>(dst) & 7u) == 0;
    for (uint64_t i = 8ull * threadIdx.x; i < a.k; i += 8ull * kThreads) {
      float v[8];
      load8(src, i, n, vec, v);
      if (s.up == 0.f) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.f;
      }
      const uint32_t lo = pack4(s(v[0]), s(v[1]), s(v[2]), s(v[3]));
      const uint32_t hi = pack4(s(v[4]), s(v[5]), s(v[6]), s(v[7]));
      if (vec_out && i + 8 <= a.k) {
        *reinterpret_cast<uint2 *>(dst + i) = make_uint2(lo, hi);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (i + e < a.k) dst[i + e] = static_cast<int8_t>((e < 4 ? lo >> (8 * e) : hi >> (8 * e - 32)) & 0xff);
      }
    }
    if (threadIdx.x == 0) a.scale[r] = s.scale;
  }
}

template <class T> cudaError_t quantize(const QuantizeArgs &a, unsigned num_sms, cudaStream_t stream) {
  const uint64_t resident = static_cast<uint64_t>(num_sms) * 8;
  auto go = [&](auto kernel, uint32_t rows_per_block) {
    const uint64_t want = (static_cast<uint64_t>(a.rows) + rows_per_block - 1) / rows_per_block;
    return launch_chained(kernel, static_cast<unsigned>(want < resident ? want : resident), kThreads, 0,
                          stream, a);
  };
  // a warp holds rows of up to 1024 values, a block rows of up to 2048 or 8192
  if (a.k <= 1024) return go(quantize_rows_kernel<T, 32, 4>, kWarps);
  if (a.k <= 2048) return go(quantize_rows_kernel<T, kThreads, 1>, 1);
  if (a.k <= 8192) return go(quantize_rows_kernel<T, kThreads, 4>, 1);
  return go(quantize_long_rows_kernel<T>, 1);
}

} // namespace

cudaError_t launch_stage(const StageArgs &a, unsigned num_sms, cudaStream_t stream) {
  if (a.count == 0) return cudaSuccess;
  uint64_t rows = 0;
  for (int i = 0; i < a.count; ++i) rows += static_cast<uint64_t>(a.op[i].batch) * a.op[i].outer;
  const uint64_t want = (rows + kWarps - 1) / kWarps, resident = static_cast<uint64_t>(num_sms) * 8;
  const unsigned grid = static_cast<unsigned>(want < 1 ? 1 : want < resident ? want : resident);
  if (a.elem_bytes == 4 && a.scale) {
    const cudaError_t e = launch_chained(largest_magnitude_kernel, kScaleRecords, kThreads, 0, stream, a);
    if (e != cudaSuccess) return e;
  }
  switch (a.elem_bytes) {
  case 1:
    return launch_chained(stage_kernel<1>, grid, kThreads, 0, stream, a);
  case 2:
    return launch_chained(stage_kernel<2>, grid, kThreads, 0, stream, a);
  default:
    return launch_chained(stage_kernel<4>, grid, kThreads, 0, stream, a);
  }
}

cudaError_t launch_quantize_rows(const QuantizeArgs &a, unsigned num_sms, cudaStream_t stream) {
  switch (static_cast<GroupedOut>(a.type)) {
  case GroupedOut::f32:
    return quantize<float>(a, num_sms, stream);
  case GroupedOut::bf16:
    return quantize<__nv_bfloat16>(a, num_sms, stream);
  default:
    return quantize<__half>(a, num_sms, stream);
  }
}

} // namespace cumpsgemm_b200
