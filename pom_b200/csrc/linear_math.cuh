// Activations of the linear operator and their derivatives ("slopes").
//
//   gelu       z Phi(z), Phi(z) = (1 + erf(z / sqrt 2)) / 2          slope Phi(z) + z exp(-z^2 / 2) / sqrt(2 pi)
//   gelu_tanh  z s(2u),  u = sqrt(2 / pi) (z + 0.044715 z^3)         slope s + z s (1 - s) 2u',  s = 1 / (1 + exp(-2u))
//   silu       z s(z)                                                slope s (1 + z (1 - s))
//   relu       max(z, 0), NaN kept                                   slope 1 for z > 0, else 0
#pragma once
#include <cuda_runtime.h>
#include "../../include/pom_b200.h"

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

// act(z) and, with SLOPE, act'(z).  FAST (bf16 results): Phi from the rational approximation 7.1.26 of Abramowitz and
// Stegun, Handbook of Mathematical Functions (1964), erfc(a) = t (a1 + t (a2 + ...)) exp(-a^2), t = 1 / (1 + p a), off by
// at most 1.5e-7, and exponentials and reciprocals of the approximate units (2 units in the last place): errors of 2^-22
// where bf16 keeps 2^-9.  The exponential serves the slope as well.  32768 x 1152 -> 4608 with slope: 397 us with erff and
// expf, FAST_TIME with these; the epilogue's instructions are what that product waits for.
template <bool SLOPE, bool FAST>
__device__ __forceinline__ float linear_act(int kind, float z, float& slope) {
  if (kind == POM_ACT_GELU) {
    float phi, e;
    if (FAST) {
      const float a = fabsf(z);
      const float t = fast_rcp(fmaf(0.2316418882f, a, 1.f));  // 0.3275911 / sqrt 2
      e = fast_exp2(-0.72134752044f * z * z);                 // exp(-z^2 / 2)
      float q = fmaf(0.5307027145f, t, -0.7265760135f);       // the five coefficients, halved
      q = fmaf(q, t, 0.7107068705f);
      q = fmaf(q, t, -0.142248368f);
      q = fmaf(q, t, 0.127414796f);
      q *= t * e;  // Phi(-|z|)
      phi = z < 0.f ? q : 1.f - q;
    } else {
      phi = 0.5f * (1.f + erff(z * 0.70710678118654752f));
      e = SLOPE ? expf(-0.5f * z * z) : 0.f;
    }
    if (SLOPE) slope = fmaf(z * 0.3989422804014327f, e, phi);
    return z * phi;
  }
  if (kind == POM_ACT_GELU_TANH || kind == POM_ACT_SILU) {
    const bool tanh = kind == POM_ACT_GELU_TANH;
    const float z2 = z * z;
    const float u = tanh ? 1.5957691216057308f * z * fmaf(0.044715f, z2, 1.f) : z;
    const float s = FAST ? fast_rcp(1.f + fast_exp2(-1.4426950408889634f * u)) : 1.f / (1.f + expf(-u));
    if (SLOPE) {
      const float du = tanh ? 1.5957691216057308f * fmaf(0.134145f, z2, 1.f) : 1.f;
      slope = s * fmaf(z * (1.f - s), du, 1.f);
    }
    return z * s;
  }
  if (kind == POM_ACT_RELU) {
    if (SLOPE) slope = z > 0.f ? 1.f : 0.f;
    return z < 0.f ? 0.f : z;
  }
  if (SLOPE) slope = 1.f;
  return z;
}

}  // namespace pomk
