// Activations that follow a matrix product, and their derivatives, in 32 bits.  An epilogue applies them to every element of a
// result, so that what they cost in instructions is what many of these products are bound by: exponential and reciprocal are single
// instructions of a relative error of 2^-22 and 2^-23, far below the 2^-9 or 2^-12 of the result's rounding.
#pragma once
#include "dfa3d_b200.h"

namespace dfa3d {

__device__ __forceinline__ float power_of_two(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float reciprocal(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 1 / (1 + exp(-z)); far below 0 exp is infinite and the reciprocal 0
__device__ __forceinline__ float sigmoid(float z) { return reciprocal(1.f + power_of_two(z * -1.4426950408889634f)); }

// The normal distribution's P(X <= z) = erfc(-z / sqrt 2) / 2 and exp(-z^2 / 2).  With t = 1 / (1 + 0.3275911 x),
// erfc(x) = exp(-x^2) (a1 t + ... + a5 t^5), |error| <= 1.5e-7, for x >= 0 (Abramowitz and Stegun, Handbook of Mathematical
// Functions, 7.1.26); on the negative side the factor exp(-x^2) keeps the tail's relative error small too.
__device__ __forceinline__ float normal_cdf(float z, float &bell) {
  bell = power_of_two(z * z * -0.72134752044448170f);
  const float t = reciprocal(fmaf(fabsf(z), 0.3275911f * 0.70710678118654752f, 1.f));
  float w = fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f);
  w = fmaf(t, w, 0.5f * 1.421413741f);
  w = fmaf(t, w, 0.5f * -0.284496736f);
  w = fmaf(t, w, 0.5f * 0.254829592f);
  w = w * t * bell;
  return z < 0.f ? w : 1.f - w;
}

template <int ACT> __device__ __forceinline__ float activate(float z) {
  if constexpr (ACT == DFA3D_ROW_RELU) return z <= 0.f ? 0.f : z;          // NaN stays
  if constexpr (ACT == DFA3D_ROW_SILU) return z * sigmoid(z);
  if constexpr (ACT == DFA3D_ROW_GELU) {
    float bell;
    return z * normal_cdf(z, bell);
  }
  return z;
}

// act(z) and d act / dz
template <int ACT> __device__ __forceinline__ void activate_both(float z, float &a, float &slope) {
  a = z;
  slope = 1.f;
  if constexpr (ACT == DFA3D_ROW_RELU) {
    a = z <= 0.f ? 0.f : z;
    slope = z <= 0.f ? 0.f : 1.f;
  }
  if constexpr (ACT == DFA3D_ROW_SILU) {
    const float s = sigmoid(z);
    a = z * s;
    slope = fmaf(a, 1.f - s, s);
  }
  if constexpr (ACT == DFA3D_ROW_GELU) {
    float bell;
    const float p = normal_cdf(z, bell);
    a = z * p;
    slope = fmaf(z * 0.39894228040143268f, bell, p);
  }
}

}  // namespace dfa3d
