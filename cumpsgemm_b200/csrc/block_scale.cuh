// Values to 8-bit floating point with one scale for a block of 128 (block_rows.cu, f8_gemm.cu).
//
// top = max |x_i|, scale = top / 448 (e4m3; e5m2: 57344), q_i = the 8-bit value nearest to x_i * 448 / top, where
// the product is rounded to FP32 and the quotient is rounded to FP32 once.  16-bit x_i have an exact product, and a
// quotient in FP32 lies on a tie between two 8-bit values only if it does unrounded, so there q_i is the nearest to
// the quotient itself.  (Multiplied with a rounded 448 / top instead, values half way between two 8-bit ones, which
// are common, go either way: 0.1 % of the norm of a product of such rows.)
// A block of zeros, or so small that its scale is 0 in FP32, has scale 0 and q = 0; one with an infinity or NaN
// has scale NaN and q = 0, so every product with it is NaN.
#pragma once
#include <cstdint>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

namespace cumpsgemm_b200 {

enum class F8Type : int { e4m3 = 0, e5m2 = 1 };

struct BlockScale {
  float scale, up, top, inverse; // up: a power of two that brings the largest near 1, times the type's largest value
  bool zero; // q is 0
  __device__ __forceinline__ BlockScale(float largest, F8Type type) {
    const float most = type == F8Type::e4m3 ? 448.f : 57344.f;
    const uint32_t e = __float_as_uint(largest) >> 23; // (largest is not negative)
    const bool none = e == 255u;
    scale = none ? __uint_as_float(0x7fffffffu) : over(largest, most, type);
    zero = none || scale == 0.f;
    // (at most 2^108, so that nothing overflows; what underflows is 0 in 8 bits)
    const float power = __uint_as_float(min(max(254u - min(e, 254u), 1u), 235u) << 23);
    top = zero ? 1.f : largest * power;
    const float about = __fdividef(1.f, top); // (one Newton step more; quotient() needs no more than that)
    inverse = __fmaf_rn(__fmaf_rn(-top, about, 1.f), about, about);
    up = power * most; // (exact)
  }
  // largest / most, rounded once.  The step that makes a product with the rounded reciprocal the rounded quotient
  // (Markstein's, with the remainder from a fused multiply-add) holds where nothing comes near the subnormals.
  static __device__ __forceinline__ float over(float largest, float most, F8Type type) {
    if (largest < 0x1p-90f) return __fdiv_rn(largest, most);
    const float r = type == F8Type::e4m3 ? 1.f / 448.f : 1.f / 57344.f, q = __fmul_rn(largest, r);
    return __fmaf_rn(__fmaf_rn(-q, most, largest), r, q);
  }
  // x * most / top: the same step.  Where the quotient is a tie between two 8-bit values, the remainder is exact, its
  // product with the reciprocal is off by 2^-22 of itself, and the sum is rounded to the tie.
  __device__ __forceinline__ float quotient(float x) const {
    const float p = __fmul_rn(x, up), q = __fmul_rn(p, inverse);
    return __fmaf_rn(__fmaf_rn(-q, top, p), inverse, q);
  }
  // The same with one factor, rounded twice: for values that are sums themselves, where no tie is meant.  Where it
  // would over- or underflow, by quotient().
  __device__ __forceinline__ bool plain(float &factor) const {
    factor = __fmul_rn(up, inverse);
    return factor > 0x1p-100f && factor < 0x1p100f;
  }
  template <F8Type TYPE>
  static __device__ __forceinline__ uint32_t four_by(float f, float x, float y, float z, float w) {
    constexpr auto kind = TYPE == F8Type::e4m3 ? __NV_E4M3 : __NV_E5M2;
    return __nv_cvt_float2_to_fp8x2(make_float2(x * f, y * f), __NV_SATFINITE, kind) |
           static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(z * f, w * f), __NV_SATFINITE, kind)) << 16;
  }
  template <F8Type TYPE> __device__ __forceinline__ uint32_t pair(float x, float y) const {
    return __nv_cvt_float2_to_fp8x2(make_float2(quotient(x), quotient(y)), __NV_SATFINITE,
                                    TYPE == F8Type::e4m3 ? __NV_E4M3 : __NV_E5M2);
  }
  template <F8Type TYPE> __device__ __forceinline__ uint32_t four(float x, float y, float z, float w) const {
    return zero ? 0u : pair<TYPE>(x, y) | pair<TYPE>(z, w) << 16;
  }
};

} // namespace cumpsgemm_b200
