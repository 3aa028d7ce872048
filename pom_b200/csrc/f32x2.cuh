// Two fp32 values per 64-bit register pair: one instruction for both, each the IEEE operation of its half.  For kernels
// that are bound by the instructions they issue.
#pragma once
#include <cuda_runtime.h>

namespace pomk {

struct F2 {
  float2 v;
  __device__ __forceinline__ F2() {}
  __device__ __forceinline__ F2(float a, float b) : v(make_float2(a, b)) {}
  __device__ __forceinline__ explicit F2(float a) : v(make_float2(a, a)) {}
};
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<unsigned long long&>(d.v))
      : "l"(reinterpret_cast<unsigned long long&>(a.v)), "l"(reinterpret_cast<unsigned long long&>(b.v)),
        "l"(reinterpret_cast<unsigned long long&>(c.v)));
  return d;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long&>(d.v))
      : "l"(reinterpret_cast<unsigned long long&>(a.v)), "l"(reinterpret_cast<unsigned long long&>(b.v)));
  return d;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<unsigned long long&>(d.v))
      : "l"(reinterpret_cast<unsigned long long&>(a.v)), "l"(reinterpret_cast<unsigned long long&>(b.v)));
  return d;
}

}  // namespace pomk
