// The activations of a gated feed-forward block, h = act(gate) * up, and their derivatives, in FP32.
//
//   silu       g p,  p = 1 / (1 + exp(-g))                    slope p + g p (1 - p)
//   gelu       g P,  P = erfc(-g / sqrt 2) / 2                slope P + g exp(-g^2 / 2) / sqrt(2 pi)
//   gelu_tanh  g (1 + tanh z) / 2 = g p,  p = 1 / (1 + exp(-2 z)),  z = sqrt(2 / pi) (g + 0.044715 g^3)
//                                                             slope p + 2 g p (1 - p) z'
//   relu       max(g, 0)                                      slope 1 above 0, else 0
//
// The forms with p and erfc lose nothing to cancellation where g is far below 0.  Where the second term of a
// slope has come to 0 it is left out, so that an infinite g (times 0) does not make it NaN.
#pragma once
#include <cuda_runtime.h>

namespace cumpsgemm_b200 {

enum class Activation : int { silu = 0, gelu = 1, gelu_tanh = 2, relu = 3 };

struct ActResult {
  float value, slope;
};

// FAST: for results of 16 or 8 bits.  exp by the approximation of 2^x, whose relative error is 2^-22 + |v| 2^-23, and
// the reciprocal to 1 unit in the last place; both are far inside the rounding that follows.  Without the forms for
// subnormals: an exp(-v) below 2^-126 counts for nothing beside 1, and where it passes 2^126 the quotient is 0 for what
// is at most 2^-126.
template <bool FAST> __device__ __forceinline__ float logistic(float v) {
  if constexpr (FAST) {
    float e, p;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v * -1.44269504088896341f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(p) : "f"(1.f + e));
    return p;
  } else {
    return 1.f / (1.f + expf(-v));
  }
}

// The slope costs nothing where it is not used.
template <Activation ACT, bool FAST> __device__ __forceinline__ ActResult activate(float g) {
  constexpr float kRootHalf = 0.707106781186547524f, kRootTwoOverPi = 0.797884560802865356f,
                  kOverRootTwoPi = 0.398942280401432678f, kCubic = 0.044715f;
  ActResult r;
  if constexpr (ACT == Activation::silu) {
    const float p = logistic<FAST>(g), q = p * (1.f - p);
    r.value = g * p;
    r.slope = q != 0.f ? fmaf(g, q, p) : p;
  } else if constexpr (ACT == Activation::gelu) {
    const float p = 0.5f * erfcf(-g * kRootHalf), e = -0.5f * g * g, q = kOverRootTwoPi * (FAST ? __expf(e) : expf(e));
    r.value = g * p;
    r.slope = q != 0.f ? fmaf(g, q, p) : p;
  } else if constexpr (ACT == Activation::gelu_tanh) {
    const float gg = g * g;
    const float p = logistic<FAST>(2.f * kRootTwoOverPi * g * fmaf(kCubic, gg, 1.f)), q = p * (1.f - p);
    r.value = g * p;
    r.slope = q != 0.f ? fmaf(2.f * g * q, kRootTwoOverPi * fmaf(3.f * kCubic, gg, 1.f), p) : p;
  } else {
    r.value = g < 0.f ? 0.f : g; // (NaN stays NaN)
    r.slope = g > 0.f ? 1.f : 0.f;
  }
  return r;
}

// g = dh up act'(gate), u = dh act(gate), of the gradient dh of act(gate) up.  OVERFLOWN (float16): gate and up were rounded,
// and an infinity stands for a sum past the type's largest value.  Such a one times nothing is nothing, and not NaN: where no
// gradient comes back (masked rows), where the activation has no slope, and where the gate is far below 0.  Anywhere
// else the gradient passes the type's largest value as well.
template <Activation ACT, bool FAST, bool OVERFLOWN>
__device__ __forceinline__ void gated_gradient(float gate, float up, float dh, float &g, float &u) {
  if constexpr (OVERFLOWN) { // (NaN stays NaN)
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(gate) : "f"(gate), "f"(-65504.f));
    const ActResult a = activate<ACT, FAST>(gate);
    float value;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(value) : "f"(a.value), "f"(3.402823466e38f));
    const float d = dh * a.slope;
    g = d == 0.f && fabsf(up) == __uint_as_float(0x7f800000u) ? 0.f : d * up;
    u = dh * value;
  } else {
    const ActResult a = activate<ACT, FAST>(gate);
    g = dh * up * a.slope;
    u = dh * a.value;
  }
}

// f(ActivationIs<a>{}): a loop asks once, and not for each of its values.
template <Activation A> struct ActivationIs {
  static constexpr Activation value = A;
};
template <class F> __device__ __forceinline__ void with_activation(int a, F &&f) {
  switch (static_cast<Activation>(a)) {
  case Activation::silu:
    return f(ActivationIs<Activation::silu>{});
  case Activation::gelu:
    return f(ActivationIs<Activation::gelu>{});
  case Activation::gelu_tanh:
    return f(ActivationIs<Activation::gelu_tanh>{});
  default:
    return f(ActivationIs<Activation::relu>{});
  }
}

} // namespace cumpsgemm_b200
