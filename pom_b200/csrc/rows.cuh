// Element access of the row-wise kernels (layer norm, linear epilogues, rotation): VEC adjacent values of one type as
// one access, kept as loaded (bf16 packed) until they are used.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <type_traits>
#include "common.cuh"
#include "ptx_sm100.cuh"

namespace pomk {

template <int BYTES>
struct RawBytes;
template <>
struct RawBytes<16> {
  using type = uint4;
};
template <>
struct RawBytes<8> {
  using type = uint2;
};
template <>
struct RawBytes<4> {
  using type = uint32_t;
};
template <>
struct RawBytes<2> {
  using type = uint16_t;
};

// VEC values of T (2 to 16 bytes, aligned to their size).
template <class T, int VEC>
struct Piece {
  static constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  using R = typename RawBytes<VEC * sizeof(T)>::type;
  union {
    R raw;
    uint32_t w[VEC * sizeof(T) >= 4 ? VEC * sizeof(T) / 4 : 1];
    uint16_t h[VEC * sizeof(T) / 2];
    float f[VEC * sizeof(T) >= 4 ? VEC * sizeof(T) / 4 : 1];
  };
  __device__ __forceinline__ void ld(const T* __restrict__ p) { raw = __ldg(reinterpret_cast<const R*>(p)); }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < static_cast<int>(VEC * sizeof(T) / 2); ++i) h[i] = 0;
  }
  __device__ __forceinline__ void st(T* __restrict__ p) const { *reinterpret_cast<R*>(p) = raw; }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (!kBf16) return f[e];
    else if constexpr (VEC == 1) return __uint_as_float(static_cast<uint32_t>(h[0]) << 16);
    else return __uint_as_float((e & 1) ? (w[e >> 1] & 0xffff0000u) : (w[e >> 1] << 16));
  }
  // rounds to nearest even
  __device__ __forceinline__ void set(const float (&v)[VEC]) {
    if constexpr (!kBf16) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] = v[e];
    } else if constexpr (VEC == 1) {
      h[0] = __bfloat16_as_ushort(__float2bfloat16_rn(v[0]));
    } else {
#pragma unroll
      for (int e = 0; e < VEC / 2; ++e) {
        const __nv_bfloat162 q = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
        w[e] = *reinterpret_cast<const uint32_t*>(&q);
      }
    }
  }
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sums of the rows of a (rows, cols) fp32 matrix of partial sums, in the type W: columns below `cut` go to out0, the
// others to out1 (either may be null).  Block = 32 columns x 32 lanes; lane l adds rows l, l + 32, ..., and the lanes are
// added in the fixed order of the shuffles: the same bits on every run.
template <class W>
__global__ void __launch_bounds__(1024) sum_rows_kernel(const float* __restrict__ partial, int rows, int cols, int cut,
                                                        W* out0, W* out1) {
  __shared__ float sm[32][33];
  griddep_wait();
  griddep_launch();
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + tx;
  float s = 0.f;
  if (c < cols)
    for (int r = ty; r < rows; r += 32) s += __ldg(partial + static_cast<long long>(r) * cols + c);
  sm[ty][tx] = s;
  __syncthreads();
  s = warp_sum(sm[tx][ty]);  // warp ty finishes column ty
  const int co = blockIdx.x * 32 + ty;
  if (tx == 0 && co < cols) {
    W* out = co < cut ? out0 : out1;
    if (out) {
      Piece<W, 1> p;
      const float v[1] = {s};
      p.set(v);
      p.st(out + (co < cut ? co : co - cut));
    }
  }
}

}  // namespace pomk

namespace pomh {

// sum_rows_kernel in the type `dtype` names.
inline int sum_rows(const float* partial, int rows, int cols, int cut, int dtype, void* out0, void* out1, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(ceil_div(cols, 32)));
  const cudaError_t e =
      dtype == POM_BF16
          ? launch_pdl(pomk::sum_rows_kernel<__nv_bfloat16>, grid, dim3(1024), 0, st, partial, rows, cols, cut,
                       static_cast<__nv_bfloat16*>(out0), static_cast<__nv_bfloat16*>(out1))
          : launch_pdl(pomk::sum_rows_kernel<float>, grid, dim3(1024), 0, st, partial, rows, cols, cut,
                       static_cast<float*>(out0), static_cast<float*>(out1));
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return POM_ERR_CUDA;
  }
  count_launch();
  return POM_OK;
}

}  // namespace pomh
