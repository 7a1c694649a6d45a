// Rows of a matrix at any address as kernels that pass over them read and write them: 16 bytes at a time,
// values in groups of eight (row_kernels.cu, block_rows.cu).
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>

namespace cumpsgemm_b200 {
namespace {

__device__ __forceinline__ bool finite(float v) {
  return (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u;
}

// A row of `bytes` bytes at any address, read 16 bytes at a time.  Where the address is no multiple of
// 16, two aligned accesses inside the row are shifted together (the second is the next lane's first,
// and comes from L1): element by element, 55 million FP32 values in odd rows took 95 us to split, and
// take 84 (5.3 TB/s).
// bytes shift .. shift + 15 of the 32 in x and y; ES divides shift
template <int ES>
__device__ __forceinline__ uint4 shifted(const uint4 &x, const uint4 &y, uint32_t shift) {
  uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
  for (int i = 0; i < 6; ++i) w[i] = shift & 8u ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) w[i] = shift & 4u ? w[i + 1] : w[i];
  if constexpr (ES < 4) {
    const uint32_t bits = (shift & 3u) * 8u;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], bits);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

struct RowReader {
  const uint8_t *p;
  uint64_t bytes;
  uint32_t shift; // p modulo 16
  __device__ __forceinline__ RowReader(const void *row, uint64_t n)
      : p(static_cast<const uint8_t *>(row)), bytes(n),
        shift(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row)) & 15u) {}
  // whether bytes at .. at + 15 can be had by aligned accesses inside the row
  __device__ __forceinline__ bool inside(uint64_t at) const {
    return at >= shift && at - shift + (shift == 0 ? 16u : 32u) <= bytes;
  }
  // For j < N the 16 bytes from at + j * step on, 0 where they are not inside.  All loads are on their way
  // before the first is looked at.  ES: bytes of an element, which divides shift; WHOLE: shift is 0; FIXED: nobody
  // writes the row while the kernel runs.
  template <int ES, bool WHOLE, bool FIXED, int N>
  __device__ __forceinline__ void load_inside(uint64_t at, uint64_t step, uint4 (&o)[N]) const {
    uint4 next[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const uint64_t from = at + j * step;
      o[j] = next[j] = make_uint4(0, 0, 0, 0);
      if (WHOLE ? from + 16 <= bytes : inside(from)) {
        const uint4 *a = reinterpret_cast<const uint4 *>(p + (WHOLE ? from : from - shift));
        o[j] = FIXED ? __ldg(a) : *a;
        if (!WHOLE && shift != 0) next[j] = FIXED ? __ldg(a + 1) : a[1];
      }
    }
    if (WHOLE || shift == 0) return;
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = shifted<ES>(o[j], next[j], shift);
  }
  // the rest of such 16 bytes: at the ends of the row, element by element
  template <int ES> __device__ __forceinline__ uint4 load_end(uint64_t at) const {
    uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
    for (uint32_t i = 0; i < 16; i += ES)
      if (at + i < bytes) {
        if (ES == 4) v[i / 4] = *reinterpret_cast<const uint32_t *>(p + at + i);
        else if (ES == 2)
          v[i / 4] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t *>(p + at + i)) << (8 * (i & 3u));
        else v[i / 4] |= static_cast<uint32_t>(p[at + i]) << (8 * (i & 3u));
      }
    return make_uint4(v[0], v[1], v[2], v[3]);
  }
  // The 16-byte pieces that are not inside are the first, where the row is not aligned, and at most three at
  // the end: piece `i` (0 .. 3) of them, or a place behind the row.
  __device__ __forceinline__ uint64_t end_piece(uint32_t i) const {
    if (i == 0) return shift == 0 ? bytes : 0;
    uint64_t first = bytes < (shift == 0 ? 16u : 32u) - shift ? 0 : (bytes + shift - (shift == 0 ? 16u : 32u)) / 16 * 16 + 16;
    if (shift != 0 && first < 16) first = 16;
    return first + 16 * (i - 1);
  }
  template <int ES, bool WHOLE, bool FIXED = true, int N>
  __device__ __forceinline__ void load(uint64_t at, uint64_t step, uint4 (&o)[N]) const {
    load_inside<ES, WHOLE, FIXED>(at, step, o);
    if constexpr (!WHOLE) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const uint64_t from = at + j * step;
        if (!inside(from) && from < bytes) o[j] = load_end<ES>(from);
      }
    }
  }
};
// Eight values of a row as they lie in memory.  The largest magnitude is taken on the bits, which are
// ordered as the values and have NaN above all of them; 16-bit types two at a time.
template <class T, bool WHOLE> struct Eight {
  static constexpr int kRegs = sizeof(T) / 2; // of 16 bytes
  uint4 raw[kRegs];
  // groups first, first + step, ... of eight values of a row
  template <bool FIXED = true, int N>
  static __device__ __forceinline__ void load(const RowReader &row, uint64_t first, uint64_t step,
                                              Eight (&v)[N]) {
    uint4 x[N * kRegs];
    if constexpr (kRegs == 1) {
      row.load<sizeof(T), WHOLE, FIXED>(first * 16, step * 16, x);
    } else {
      uint4 lo[N], hi[N];
      row.load<sizeof(T), WHOLE, FIXED>(first * 32, step * 32, lo);
      row.load<sizeof(T), WHOLE, FIXED>(first * 32 + 16, step * 32, hi);
#pragma unroll
      for (int j = 0; j < N; ++j) x[2 * j] = lo[j], x[2 * j + 1] = hi[j];
    }
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
      for (int i = 0; i < kRegs; ++i) v[j].raw[i] = x[j * kRegs + i];
  }
  __device__ __forceinline__ uint32_t largest(uint32_t top) const {
#pragma unroll
    for (int i = 0; i < kRegs; ++i) {
      const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        top = sizeof(T) == 4 ? max(top, w[j] & 0x7fffffffu) : __vmaxu2(top, w[j] & 0x7fff7fffu);
    }
    return top;
  }
  __device__ __forceinline__ void values(float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < kRegs; ++i) {
      const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 4) v[4 * i + j] = __uint_as_float(w[j]);
        else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
          v[2 * j] = __uint_as_float(w[j] << 16);
          v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        } else {
          const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[j]));
          v[2 * j] = f.x;
          v[2 * j + 1] = f.y;
        }
      }
    }
  }
};
// the largest magnitude itself, from the bits of a whole warp's threads
template <class T> __device__ __forceinline__ uint32_t warp_largest(uint32_t top) {
  if constexpr (sizeof(T) == 2) top = max(top & 0xffffu, top >> 16);
  return __reduce_max_sync(0xffffffffu, top);
}
template <class T> __device__ __forceinline__ float value_of(uint32_t bits) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(bits);
  else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __uint_as_float(bits << 16);
  else return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
}
__device__ __forceinline__ void store_eight(int8_t *row, uint64_t i, uint32_t k, uint2 q) {
  int8_t *at = row + i;
  if ((reinterpret_cast<uintptr_t>(row) & 7u) == 0 && i + 8 <= k) {
    *reinterpret_cast<uint2 *>(at) = q;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (i + e < k) at[e] = static_cast<int8_t>((e < 4 ? q.x >> (8 * e) : q.y >> (8 * e - 32)) & 0xffu);
  }
}
} // namespace
} // namespace cumpsgemm_b200
