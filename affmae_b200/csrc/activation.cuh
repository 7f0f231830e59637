// Activations of the matrix product's epilogue and their derivatives, fp32.
#pragma once

#include "common.cuh"

namespace affb {


__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// Phi(-a) of the normal distribution for a >= 0 as 2^p(a): log2 Phi(-a) is
// close to a parabola, and the degree-8 polynomial below (weighted least
// squares on [0, 8], weight Phi(-a) max(1, a)) leaves errors of 1.9e-7 in Phi
// and 1.7e-7 in a Phi, and a relative error of Phi below 2e-3 down to Phi(-8);
// the leading coefficient is negative, so the tail goes to 0.  One exponential
// and 8 FMAs, against erff's branches.
__device__ __forceinline__ float normal_tail(float a) {
  float p = -2.51915651e-07f;
  p = fmaf(p, a, 4.51663482e-06f);
  p = fmaf(p, a, -2.38722357e-08f);
  p = fmaf(p, a, -0.000637269346f);
  p = fmaf(p, a, 0.00777910277f);
  p = fmaf(p, a, -0.0530270971f);
  p = fmaf(p, a, -0.459024668f);
  p = fmaf(p, a, -1.15112805f);
  p = fmaf(p, a, -0.999999583f);
  return exp2_approx(p);
}

constexpr float LOG2E = 1.4426950408889634f;

// Two fp32 values in one register pair: the additions, products and FMAs of
// sm_100 on pairs issue once for both.
using pair_t = unsigned long long;
__device__ __forceinline__ pair_t pack2(float a, float b) {
  pair_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(pair_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ pair_t add2(pair_t a, pair_t b) {
  pair_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ pair_t mul2(pair_t a, pair_t b) {
  pair_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ pair_t fma2(pair_t a, pair_t b, pair_t c) {
  pair_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ pair_t both(float v) { return pack2(v, v); }

template <int ACT>
__device__ __forceinline__ float activate(float z) {
  if constexpr (ACT == AFFB_ACT_RELU) {
    return max_nan(z, 0.f);
  } else if constexpr (ACT == AFFB_ACT_GELU) {
    // z Phi(z) = max(z, 0) - |z| Phi(-|z|); the clamp keeps inf * 0 out
    const float a = min_nan(fabsf(z), 64.f);
    return fmaf(-a, normal_tail(a), fmaxf(z, 0.f));
  } else if constexpr (ACT == AFFB_ACT_SILU) {
    return __fdividef(z, 1.f + exp2_approx(-LOG2E * z));
  } else {
    return z;
  }
}

// activate() of two values, the polynomial of GELU on pairs.
template <int ACT>
__device__ __forceinline__ void activate_pair(float& x, float& y) {
  if constexpr (ACT == AFFB_ACT_GELU) {
    const float ax = min_nan(fabsf(x), 64.f), ay = min_nan(fabsf(y), 64.f);
    const pair_t a = pack2(ax, ay);
    pair_t p = both(-2.51915651e-07f);
    p = fma2(p, a, both(4.51663482e-06f));
    p = fma2(p, a, both(-2.38722357e-08f));
    p = fma2(p, a, both(-0.000637269346f));
    p = fma2(p, a, both(0.00777910277f));
    p = fma2(p, a, both(-0.0530270971f));
    p = fma2(p, a, both(-0.459024668f));
    p = fma2(p, a, both(-1.15112805f));
    p = fma2(p, a, both(-0.999999583f));
    float px, py;
    unpack2(p, px, py);
    x = fmaf(-ax, exp2_approx(px), fmaxf(x, 0.f));
    y = fmaf(-ay, exp2_approx(py), fmaxf(y, 0.f));
  } else {
    x = activate<ACT>(x);
    y = activate<ACT>(y);
  }
}

template <int ACT>
__device__ __forceinline__ float activate_grad(float z) {  // not of ReLU: see through_grad
  if constexpr (ACT == AFFB_ACT_GELU) {
    const float a = min_nan(fabsf(z), 64.f);
    const float t = normal_tail(a);
    // Phi(z) + z phi(z)
    const float pdf = 0.3989422804014327f * exp2_approx(-0.5f * LOG2E * a * a);
    return fmaf(copysignf(a, z), pdf, z > 0.f ? 1.f - t : t);
  } else if constexpr (ACT == AFFB_ACT_SILU) {
    const float c = max_nan(min_nan(z, 64.f), -64.f);  // keeps inf * 0 out
    const float s = __fdividef(1.f, 1.f + exp2_approx(-LOG2E * c));
    return s * fmaf(c, 1.f - s, 1.f);
  } else {
    return 1.f;
  }
}

// The gradient d of act(z) as that of z.  ReLU selects: an infinite or NaN
// gradient of a value it has cut off is no gradient.
template <int ACT>
__device__ __forceinline__ float through_grad(float d, float z) {
  if constexpr (ACT == AFFB_ACT_RELU) return z <= 0.f ? 0.f : d;
  return d * activate_grad<ACT>(z);
}

}  // namespace affb
