// Activations that follow a matrix product, and their derivatives, in 32 bits, two elements at a time.  An epilogue applies them to
// every element of a result, and what they cost in instructions is what many of these products are bound by.  So: products and sums of
// two elements are one instruction; exponential and reciprocal are single instructions of a relative error of 2^-22 and 2^-23, far
// below the 2^-9 or 2^-12 of the result's rounding; and since an SM has a quarter as many units for those two, two reciprocals are one,
// 1 / a = b / (a b).
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
__device__ __forceinline__ float no_less(float x, float least) {      // NaN stays
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(x), "f"(least));
  return y;
}

struct Two {
  float x, y;
};
__device__ __forceinline__ Two both(float c) { return {c, c}; }
__device__ __forceinline__ Two operator+(Two a, Two b) {
  asm("{\n.reg .b64 p, q;\nmov.b64 p, {%0, %1};\nmov.b64 q, {%2, %3};\nadd.rn.f32x2 p, p, q;\nmov.b64 {%0, %1}, p;\n}"
      : "+f"(a.x), "+f"(a.y)
      : "f"(b.x), "f"(b.y));
  return a;
}
__device__ __forceinline__ Two operator*(Two a, Two b) {
  asm("{\n.reg .b64 p, q;\nmov.b64 p, {%0, %1};\nmov.b64 q, {%2, %3};\nmul.rn.f32x2 p, p, q;\nmov.b64 {%0, %1}, p;\n}"
      : "+f"(a.x), "+f"(a.y)
      : "f"(b.x), "f"(b.y));
  return a;
}
__device__ __forceinline__ Two times_plus(Two a, Two b, Two c) {      // a b + c
  asm("{\n.reg .b64 p, q, r;\nmov.b64 p, {%0, %1};\nmov.b64 q, {%2, %3};\nmov.b64 r, {%4, %5};\nfma.rn.f32x2 p, p, q, r;\nmov.b64 {%0, "
      "%1}, p;\n}"
      : "+f"(a.x), "+f"(a.y)
      : "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return a;
}
__device__ __forceinline__ Two power_of_two(Two a) { return {power_of_two(a.x), power_of_two(a.y)}; }
__device__ __forceinline__ Two reciprocal(Two a) {      // of numbers from 1 to 2^61
  const float r = reciprocal(a.x * a.y);
  return {r * a.y, r * a.x};
}

// e^z / (1 + e^z), 1 from 2^60 on: on the negative side as right relative to itself as e^z is, down to where 32 bits end
__device__ __forceinline__ Two sigmoid(Two z) {
  Two q = z * both(1.4426950408889634f);
  q = {fminf(q.x, 60.f), fminf(q.y, 60.f)};
  const Two e = power_of_two(q);
  return e * reciprocal(e + both(1.f));
}
// z as far as it counts: z sigmoid(z) is 0 at -infinity
__device__ __forceinline__ Two counted(Two z) { return {no_less(z.x, -1e30f), no_less(z.y, -1e30f)}; }

// The normal distribution's P(X <= z) and exp(-z^2 / 2).  P(X <= -|z|) = exp(-z^2 / 2) R(|z|) with R(|z|) = erfcx(|z| / sqrt 2) / 2, which
// falls as 1 / |z| and is a polynomial of t = 1 / (1 + 0.365 |z| / sqrt 2) without a constant term: seven terms, fitted to the
// definition on 0 <= |z| <= 13.5 by a linear program over 1200 points so that the probability is off by at most 3e-8 and by at most
// 2^-18.7 of itself.  So the tail is right too: with the roundings to 4e-6 of itself up to |z| = 6 and to 1e-5 up to 13, where 32 bits
// end; a bound of the first kind alone leaves 1 % at 8.
__device__ __forceinline__ Two normal_cdf(Two z, Two &bell) {
  bell = power_of_two(z * z * both(-0.72134752044448170f));
  const Two far{fminf(fabsf(z.x), 1e8f), fminf(fabsf(z.y), 1e8f)};
  const Two t = reciprocal(times_plus(far, both(0.365f * 0.70710678118654752f), both(1.f)));
  Two w = times_plus(t, both(-0.076127111f), both(0.247021068f));
  w = times_plus(t, w, both(-0.129819675f));
  w = times_plus(t, w, both(0.181564439f));
  w = times_plus(t, w, both(0.067287249f));
  w = times_plus(t, w, both(0.107386443f));
  w = times_plus(t, w, both(0.102687557f));
  w = w * (t * bell);
  const Two v = times_plus(w, both(-1.f), both(1.f));
  return {z.x < 0.f ? w.x : v.x, z.y < 0.f ? w.y : v.y};
}

template <int ACT> __device__ __forceinline__ Two activate(Two z) {
  if constexpr (ACT == DFA3D_ROW_RELU) return {z.x <= 0.f ? 0.f : z.x, z.y <= 0.f ? 0.f : z.y};          // NaN stays
  if constexpr (ACT == DFA3D_ROW_SILU) return counted(z) * sigmoid(z);
  if constexpr (ACT == DFA3D_ROW_GELU) {
    Two bell;
    return z * normal_cdf(z, bell);
  }
  return z;
}

// act(z) and d act / dz
template <int ACT> __device__ __forceinline__ void activate_both(Two z, Two &a, Two &slope) {
  a = z;
  slope = both(1.f);
  if constexpr (ACT == DFA3D_ROW_RELU) {
    a = activate<ACT>(z);
    slope = {z.x <= 0.f ? 0.f : 1.f, z.y <= 0.f ? 0.f : 1.f};
  }
  if constexpr (ACT == DFA3D_ROW_SILU) {
    const Two s = sigmoid(z);
    a = counted(z) * s;
    slope = times_plus(a, times_plus(s, both(-1.f), both(1.f)), s);
  }
  if constexpr (ACT == DFA3D_ROW_GELU) {
    Two bell;
    const Two p = normal_cdf(z, bell);
    a = z * p;
    slope = times_plus(z * both(0.39894228040143268f), bell, p);
  }
}

}  // namespace dfa3d
