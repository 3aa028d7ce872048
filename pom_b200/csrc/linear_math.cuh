// Activations of the linear operator and their derivatives ("slopes").
//
//   gelu       z Phi(z), Phi(z) = erfc(-z / sqrt 2) / 2              slope Phi(z) + z exp(-z^2 / 2) / sqrt(2 pi)
//   gelu_tanh  z s(2u),  u = sqrt(2 / pi) (z + 0.044715 z^3)         slope s + z s (1 - s) 2u',  s = 1 / (1 + exp(-2u))
//   silu       z s(z)                                                slope s (1 + z (1 - s))
//   relu       max(z, 0), NaN kept                                   slope 1 for z > 0, else 0
//
// gelu's values vanish like exp(-z^2 / 2) far below 0 and are wanted to their last digit there too, so Phi of a negative z is
// formed as itself and not as 1 less something: float32 takes erfc (errors relative to the value of a few 2^-24 and z^2 2^-24,
// what the exponent's rounding leaves; 4079 x 4608 slopes take 63 us instead of 49 with erf).
//
// FAST (bf16 results): Phi(-a) exp(a^2 / 2) is smooth and falls like 1 / a, so it is a polynomial of degree 6 without a
// constant term in t = 1 / (1 + p a): p and the six coefficients make the largest relative error over 0 <= a <= 13.3 smallest
// (weighted least squares, the weights raised where the error is large until it is the same at all its peaks), 3.6e-6.
// With exponentials and reciprocals of the approximate units the relative error is at most 4.3e-6 (2^-17.8) above z = -4 and
// 1.2e-5 (2^-16.3) down to -13.2, below which exp(-z^2 / 2) is no normal number and the result 0; bf16 keeps 2^-8.  gelu, which
// is the default of most feed-forward blocks, works on packed pairs.
#pragma once
#include <cuda_runtime.h>
#include "../../include/pom_b200.h"
#include "f32x2.cuh"

namespace pomk {

__device__ __forceinline__ float fast_rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float fast_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Phi(z) and e = exp(-z^2 / 2).
__device__ __forceinline__ F2 gelu_phi2(F2 z, F2& e) {
  const F2 d = fma2(F2(fabsf(z.v.x), fabsf(z.v.y)), F2(0.307445f), F2(1.f));
  const F2 t(fast_rcp(d.v.x), fast_rcp(d.v.y));
  const F2 w = mul2(mul2(z, F2(-0.72134752044f)), z);
  e = F2(fast_exp2(w.v.x), fast_exp2(w.v.y));
  F2 q = fma2(F2(-0.0759885991f), t, F2(0.192621113f));
  q = fma2(q, t, F2(0.00437823325f));
  q = fma2(q, t, F2(0.137688858f));
  q = fma2(q, t, F2(0.118373599f));
  q = fma2(q, t, F2(0.122924995f));
  q = mul2(q, mul2(t, e));  // Phi(-|z|)
  const F2 up = fma2(q, F2(-1.f), F2(1.f));
  return F2(z.v.x < 0.f ? q.v.x : up.v.x, z.v.y < 0.f ? q.v.y : up.v.y);
}

template <bool FAST>
__device__ __forceinline__ float linear_sigmoid(float u) {
  return FAST ? fast_rcp(1.f + fast_exp2(-1.4426950408889634f * u)) : 1.f / (1.f + expf(-u));
}

template <bool FAST>
__device__ __forceinline__ F2 linear_act2(int kind, F2 z) {
  if (kind == POM_ACT_GELU && FAST) {
    F2 e;
    return mul2(z, gelu_phi2(z, e));
  }
  auto one = [&](float x) {
    if (kind == POM_ACT_GELU) return x * (0.5f * erfcf(x * -0.70710678118654752f));
    if (kind == POM_ACT_GELU_TANH) return x * linear_sigmoid<FAST>(1.5957691216057308f * x * fmaf(0.044715f, x * x, 1.f));
    if (kind == POM_ACT_SILU) return x * linear_sigmoid<FAST>(x);
    if (kind == POM_ACT_RELU) return x < 0.f ? 0.f : x;
    return x;
  };
  return F2(one(z.v.x), one(z.v.y));
}

template <bool FAST>
__device__ __forceinline__ F2 linear_slope2(int kind, F2 z) {
  if (kind == POM_ACT_GELU && FAST) {
    F2 e;
    const F2 phi = gelu_phi2(z, e);
    return fma2(mul2(z, F2(0.3989422804014327f)), e, phi);
  }
  auto one = [&](float x) {
    if (kind == POM_ACT_GELU)
      return fmaf(x * 0.3989422804014327f, expf(-0.5f * x * x), 0.5f * erfcf(x * -0.70710678118654752f));
    if (kind == POM_ACT_GELU_TANH) {
      // beyond +-16 the slope is 1 or 0 to the last bit, and x^2 of far values would overflow into 0 * inf (NaN passes)
      x = x > 16.f ? 16.f : x < -16.f ? -16.f : x;
      const float x2 = x * x, s = linear_sigmoid<FAST>(1.5957691216057308f * x * fmaf(0.044715f, x2, 1.f));
      return s * fmaf(x * (1.f - s), 1.5957691216057308f * fmaf(0.134145f, x2, 1.f), 1.f);
    }
    if (kind == POM_ACT_SILU) {
      const float s = linear_sigmoid<FAST>(x);
      return s * fmaf(x, 1.f - s, 1.f);
    }
    if (kind == POM_ACT_RELU) return x > 0.f ? 1.f : 0.f;
    return 1.f;
  };
  return F2(one(z.v.x), one(z.v.y));
}

template <bool FAST>
__device__ __forceinline__ float linear_act(int kind, float z) {
  return linear_act2<FAST>(kind, F2(z, 0.f)).v.x;
}

}  // namespace pomk
