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

template <bool SLOPE>
__device__ __forceinline__ float linear_act(int kind, float z, float& slope) {
  if (kind == POM_ACT_GELU) {
    const float phi = 0.5f * (1.f + erff(z * 0.70710678118654752f));
    if (SLOPE) slope = fmaf(z * 0.3989422804014327f, expf(-0.5f * z * z), phi);
    return z * phi;
  }
  if (kind == POM_ACT_GELU_TANH) {
    const float z2 = z * z;
    const float s = 1.f / (1.f + expf(-1.5957691216057308f * z * fmaf(0.044715f, z2, 1.f)));
    if (SLOPE) slope = fmaf(z * s * (1.f - s), 1.5957691216057308f * fmaf(0.134145f, z2, 1.f), s);
    return z * s;
  }
  if (kind == POM_ACT_SILU) {
    const float s = 1.f / (1.f + expf(-z));
    if (SLOPE) slope = s * fmaf(z, 1.f - s, 1.f);
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
