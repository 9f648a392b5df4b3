// The activations of the gated product c = act(g) * u and their derivatives, in fp32.
//
// Each is written so that nothing cancels and nothing is infinite times zero for a finite g:
//   silu       g s(g), s the logistic function;                       d = s (1 + g (1 - s))
//   gelu       g P(g), P(g) = erfc(-g / sqrt 2) / 2 (the erf form loses the negative tail);
//                                                                     d = P + g exp(-g^2 / 2) / sqrt(2 pi)
//   gelu_tanh  g (1 + tanh z) / 2 = g s(2 z), z = sqrt(2 / pi) (g + 0.044715 g^3);
//                                                                     d = s + g s (1 - s) 2 z'
//   relu       max(g, 0), NaN kept;                                   d = 1 for g > 0, else 0
// At the infinities they are their limits: 0 with slope 0 at -infinity, infinite with slope 1 at +infinity.  The backward pass
// sees g as the forward pass kept it, in 16 bits, where a product below -65504 is -infinity in fp16.
#pragma once

#include <cfloat>

#include "sm100_ptx.cuh"

namespace beam {

enum Activation : int { kActSilu = 0, kActGelu = 1, kActGeluTanh = 2, kActRelu = 3 };

// 1 / (1 + exp(-x)).  exp overflows to infinity for x < -88.7 and the reciprocal is then 0; the approximate reciprocal (off by a
// step at most) keeps subnormal results, which __fdividef flushes for divisors above 2^126.
__device__ __forceinline__ float logistic(float x) {
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.f + __expf(-x)));
  return r;
}

constexpr float kSqrtHalf = 0.70710678118654752f;
constexpr float kInvSqrt2Pi = 0.39894228040143268f;
constexpr float kTwoSqrt2OverPi = 1.5957691216057308f;  // 2 sqrt(2 / pi)
constexpr float kGeluCubic = 0.044715f;

// The larger and the smaller of two numbers; a NaN stays one.
__device__ __forceinline__ float max_nan(float x, float y) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float min_nan(float x, float y) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}

template <int kAct>
__device__ __forceinline__ float act_value(float g) {
  if constexpr (kAct != kActRelu) g = max_nan(g, -FLT_MAX);  // where all are 0 already
  if constexpr (kAct == kActSilu) {
    return g * logistic(g);
  } else if constexpr (kAct == kActGelu) {
    return 0.5f * g * erfcf(-g * kSqrtHalf);
  } else if constexpr (kAct == kActGeluTanh) {
    return g * logistic(kTwoSqrt2OverPi * g * (1.f + kGeluCubic * g * g));
  } else {
    return max_nan(g, 0.f);
  }
}

// act(g) and act'(g) together.
template <int kAct>
__device__ __forceinline__ float2 act_value_slope(float kept) {
  const float v = max_nan(kept, -FLT_MAX);  // for the value
  const float g = min_nan(v, FLT_MAX);      // for the slope, which has its limits at the largest finite numbers
  if constexpr (kAct == kActSilu) {
    const float s = logistic(g);
    return make_float2(v * s, s * (1.f + g * (1.f - s)));
  } else if constexpr (kAct == kActGelu) {
    const float p = 0.5f * erfcf(-g * kSqrtHalf);
    return make_float2(v * p, p + g * __expf(-0.5f * g * g) * kInvSqrt2Pi);
  } else if constexpr (kAct == kActGeluTanh) {
    const float gg = kGeluCubic * g * g;
    const float s = logistic(kTwoSqrt2OverPi * g * (1.f + gg));
    const float curve = s * (1.f - s);  // exactly 0 for large |g|, where g * z' may overflow
    const float bend = curve > 0.f ? curve * g * kTwoSqrt2OverPi * (1.f + 3.f * gg) : 0.f;
    return make_float2(v * s, s + bend);
  } else {
    return make_float2(max_nan(v, 0.f), v > 0.f ? 1.f : 0.f);
  }
}

}  // namespace beam
