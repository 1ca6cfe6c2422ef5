// Activations of the row operators that follow a matrix product, and their derivatives, in 32 bits.
#pragma once
#include "dfa3d_b200.h"

namespace dfa3d {

// 1 / (1 + exp(-z)): exp overflows to infinity below -88, where the quotient is 0 as it should be
__device__ __forceinline__ float sigmoid(float z) { return __fdividef(1.f, 1.f + __expf(-z)); }

__device__ __forceinline__ float half_erfc(float z) { return 0.5f + 0.5f * erff(z * 0.70710678118654752f); }

template <int ACT> __device__ __forceinline__ float activate(float z) {
  if constexpr (ACT == DFA3D_ROW_RELU) return z <= 0.f ? 0.f : z;          // NaN stays
  if constexpr (ACT == DFA3D_ROW_SILU) return z * sigmoid(z);
  if constexpr (ACT == DFA3D_ROW_GELU) return z * half_erfc(z);
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
    slope = s + a * (1.f - s);
  }
  if constexpr (ACT == DFA3D_ROW_GELU) {
    const float p = half_erfc(z);
    a = z * p;
    slope = p + z * 0.39894228040143268f * __expf(-0.5f * z * z);
  }
}

}  // namespace dfa3d
