// The linear operator: y = act(x W^T + bias) + residual, and its backward pass.
//
//   forward   z = x W^T + bias (kept for a backward pass), y = act(z) + residual
//   backward  dz = dy act'(z);  dx = dz W;  dW = dz^T x;  dbias = sum of dz over the rows;  dresidual = dy
//
// bf16, many rows: the tcgen05 GEMM engine with EpiLinear, or, where that leaves SMs idle, clusters that share a tile
// (gemm_cluster.cuh).  Few rows: linear_few_*_kernel, which reads the weight once and spreads it over all SMs.
// float32 with more rows: the products of pom_gemm_f32_planes or pom_gemm_f32, and linear_epilogue_kernel.
//
// Sums are fp32; nothing here is summed by atomics, so a call gives the same bits every time.
#include "epilogues_linear.cuh"
#include "gemm_cluster.cuh"
#include "gemm_launch.cuh"
#include "rows.cuh"

using namespace pomk;
using namespace pomh;

namespace {

struct FewDev {
  const void *x, *w, *bias, *residual;  // an absent bias or residual: an address that may be read (see readable)
  void *y, *z;  // z (contiguous) or null
  long long ldx, ldw, ldr, ldy;
  int M, N, K, act, bias_f32;
  int has_bias, has_residual;
};

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float few_bias(const FewDev& a, int n) {
  return a.bias_f32 ? __ldg(static_cast<const float*>(a.bias) + n)
                    : __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(a.bias) + n));
}

// bias, activation, residual and stores of one output value of the few-row kernels.  Every thread of the block's outputs
// comes here: the loads stand behind no condition and read addresses that exist (row and n inside the output; an operand that is
// not there is read at the first value of x, see readable), only the stores are left out where !in.
//
// With `if (a.bias)` and `if (m < M)` in front of them, the instances whose threads finish two outputs of one column
// (MT = NT = 2) faulted at an unmapped address when there was no bias and rows were missing (20 x 1016 -> 4056): the load of the
// bias, the same for both outputs, was made outside its conditions.
template <class T>
__device__ __forceinline__ void few_finish(const FewDev& a, int row, int n, bool in, float z) {
  Piece<T, 1> p;
  const float b = few_bias(a, a.has_bias ? n : 0);
  Piece<T, 1> r;
  r.ld(static_cast<const T*>(a.residual) + (a.has_residual ? row * a.ldr + n : 0));
  z = a.has_bias ? z + b : z;
  float v[1] = {linear_act<Piece<T, 1>::kBf16>(a.act, z)};
  v[0] = a.has_residual ? v[0] + r.get(0) : v[0];
  if (!in) return;
  if (a.z) {
    const float k[1] = {z};
    p.set(k);
    p.st(static_cast<T*>(a.z) + static_cast<long long>(row) * a.N + n);
  }
  p.set(v);
  p.st(static_cast<T*>(a.y) + row * a.ldy + n);
}

constexpr int kFewWarps = 8;

// Bound by the trip to the weight, not by its bytes: 1152 -> 4608 (10.6 MB) takes 8 us from HBM at one row and 10 at 32,
// 4608 -> 1152 12.3 at one.  The tensor cores' rate does not matter, so mma.sync, which takes its operands from registers, is enough.
// The operands are read without conditions, from the last row or piece where there is none, and zeroed afterwards: the loads of
// all pieces are in flight together (behind conditions 4608 -> 1152 took 16.4 us), and none can leave its operand.
//
// Up to 16 * MT rows.  A block owns 8 * NT output columns and reads their weight rows once; its warps take 32-long pieces
// of K in turn.  Lane (g, t) holds 8 adjacent k of row g of every operand, piece t: which k of the piece the matrix
// instruction takes for which of its own k does not matter, as long as both operands agree, so the 16 bytes a lane loads
// are two instructions' fragments as they are.
template <int MT, int NT>
__global__ void __launch_bounds__(32 * kFewWarps) linear_few_bf16_kernel(const FewDev a) {
  constexpr int U = MT == 1 ? 4 : 2;  // pieces in flight
  __shared__ float red[kFewWarps][16 * MT][8 * NT + 1];
  griddep_wait();
  griddep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * 8 * NT;
  const __nv_bfloat16* w = static_cast<const __nv_bfloat16*>(a.w);
  const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(a.x);
  float c[MT][NT][4];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) c[i][j][e] = 0.f;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  for (int kc = warp * 32; kc < a.K; kc += 32 * kFewWarps * U) {
    uint4 wv[U][NT], xv[U][MT][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = kc + u * 32 * kFewWarps + t * 8;
      const bool ok = k < a.K;  // K is a multiple of 8
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int n = n0 + j * 8 + g;
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(w + min(n, a.N - 1) * a.ldw + min(k, a.K - 8)));
        wv[u][j] = ok && n < a.N ? v : zero;
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int m = i * 16 + h * 8 + g;
          const uint4 v = __ldg(reinterpret_cast<const uint4*>(x + min(m, a.M - 1) * a.ldx + min(k, a.K - 8)));
          xv[u][i][h] = ok && m < a.M ? v : zero;
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          mma_bf16(c[i][j], xv[u][i][0].x, xv[u][i][1].x, xv[u][i][0].y, xv[u][i][1].y, wv[u][j].x, wv[u][j].y);
          mma_bf16(c[i][j], xv[u][i][0].z, xv[u][i][1].z, xv[u][i][0].w, xv[u][i][1].w, wv[u][j].z, wv[u][j].w);
        }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      red[warp][i * 16 + g][j * 8 + 2 * t] = c[i][j][0];
      red[warp][i * 16 + g][j * 8 + 2 * t + 1] = c[i][j][1];
      red[warp][i * 16 + g + 8][j * 8 + 2 * t] = c[i][j][2];
      red[warp][i * 16 + g + 8][j * 8 + 2 * t + 1] = c[i][j][3];
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * MT * 8 * NT; i += 32 * kFewWarps) {
    const int m = i / (8 * NT), n = i - m * (8 * NT);
    float z = 0.f;
#pragma unroll
    for (int q = 0; q < kFewWarps; ++q) z += red[q][m][n];
    few_finish<__nv_bfloat16>(a, min(m, a.M - 1), min(n0 + n, a.N - 1), m < a.M && n0 + n < a.N, z);
  }
}

// float32, up to MR rows: a block owns 8 columns, lane (ng, kq) the 4 adjacent k of piece kq for columns ng and ng + 4.
template <int MR>
__global__ void __launch_bounds__(32 * kFewWarps) linear_few_f32_kernel(const FewDev a) {
  constexpr int U = MR <= 4 ? 4 : 2;
  __shared__ float red[kFewWarps][MR][8];
  griddep_wait();
  griddep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, kq = lane & 7, ng = lane >> 3;
  const int n0 = blockIdx.x * 8;
  const float* w = static_cast<const float*>(a.w);
  const float* x = static_cast<const float*>(a.x);
  float c[MR][2];
#pragma unroll
  for (int m = 0; m < MR; ++m) c[m][0] = c[m][1] = 0.f;
  const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int kc = warp * 32; kc < a.K; kc += 32 * kFewWarps * U) {
    float4 wv[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = kc + u * 32 * kFewWarps + kq * 4;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int n = n0 + ng + 4 * j;
        wv[u][j] = k < a.K && n < a.N ? __ldg(reinterpret_cast<const float4*>(w + n * a.ldw + k)) : zero;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = kc + u * 32 * kFewWarps + kq * 4;
#pragma unroll
      for (int m = 0; m < MR; ++m) {
        const float4 v = k < a.K && m < a.M ? __ldg(reinterpret_cast<const float4*>(x + m * a.ldx + k)) : zero;
#pragma unroll
        for (int j = 0; j < 2; ++j)
          c[m][j] = fmaf(v.w, wv[u][j].w, fmaf(v.z, wv[u][j].z, fmaf(v.y, wv[u][j].y, fmaf(v.x, wv[u][j].x, c[m][j]))));
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int o = 4; o; o >>= 1) c[m][j] += __shfl_xor_sync(0xffffffffu, c[m][j], o);
      if (kq == 0) red[warp][m][ng + 4 * j] = c[m][j];
    }
  __syncthreads();
  for (int i = threadIdx.x; i < MR * 8; i += 32 * kFewWarps) {
    const int m = i >> 3, n = i & 7;
    float z = 0.f;
#pragma unroll
    for (int q = 0; q < kFewWarps; ++q) z += red[q][m][n];
    few_finish<float>(a, min(m, a.M - 1), min(n0 + n, a.N - 1), m < a.M && n0 + n < a.N, z);
  }
}

// y = act(z + bias) + residual over (M, N), z the sum of `slabs` fp32 matrices in their order; y may be the one slab.
// VEC adjacent columns per thread.
template <class T, int VEC>
__global__ void __launch_bounds__(256) linear_epilogue_kernel(const FewDev a, const float* z, long long ldz, int slabs,
                                                              long long M) {
  griddep_wait();
  griddep_launch();
  const int per_row = a.N / VEC;
  const long long total = M * per_row, each = M * ldz;
  const bool wide_bias = a.has_bias && !(reinterpret_cast<uintptr_t>(a.bias) & 15);
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const long long r = total <= 0x7fffffff ? static_cast<unsigned>(i) / static_cast<unsigned>(per_row) : i / per_row;
    const int c = static_cast<int>(i - r * per_row) * VEC;
    Piece<float, VEC> in;
    Piece<T, VEC> q;
    // may be y: no read-only path
    in.raw = *reinterpret_cast<const typename Piece<float, VEC>::R*>(z + r * ldz + c);
    float v[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = in.get(e);
    for (int k = 1; k < slabs; k += 3) {  // three in flight
      Piece<float, VEC> more[3];
#pragma unroll
      for (int q = 0; q < 3; ++q)
        if (k + q < slabs) more[q].ld(z + (k + q) * each + r * ldz + c);
#pragma unroll
      for (int q = 0; q < 3; ++q)
        if (k + q < slabs) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) v[e] += more[q].get(e);
        }
    }
    if (wide_bias) {
      if (a.bias_f32) {
        in.ld(static_cast<const float*>(a.bias) + c);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] += in.get(e);
      } else {
        Piece<__nv_bfloat16, VEC> b;
        b.ld(static_cast<const __nv_bfloat16*>(a.bias) + c);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] += b.get(e);
      }
    } else if (a.has_bias) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] += few_bias(a, c + e);
    }
    if (a.z) {
      q.set(v);
      q.st(static_cast<T*>(a.z) + r * a.N + c);
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = linear_act<Piece<T, 1>::kBf16>(a.act, v[e]);
    if (a.has_residual) {
      q.ld(static_cast<const T*>(a.residual) + r * a.ldr + c);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] += q.get(e);
    }
    q.set(v);
    q.st(static_cast<T*>(a.y) + r * a.ldy + c);
  }
}

// One pass, bound by HBM: 32768 x 4608 bf16 with gelu 148 to 152 us (906 MB, 6.1 TB/s), where a copy would take 138.
// dz = dy act'(z) (ACT none: dz = dy, which is not written) and the column sums of dz over the block's rows.
// Block = 32 column lanes of VEC columns x 8 row lanes; grid = (column blocks, row chunks).  bf16 comes in whole 16-byte pieces
// (the products behind it want that anyway), float32 also in single values.
template <class T, int VEC, int ACT>
__global__ void __launch_bounds__(256) linear_dz_kernel(const T* __restrict__ dy, long long ld_dy, const T* __restrict__ z,
                                                        T* __restrict__ dz, float* __restrict__ partial, long long M, int N,
                                                        int chunk) {
  constexpr bool kFast = Piece<T, 1>::kBf16;
  __shared__ float sm[8][32 * VEC + 1];
  griddep_wait();
  griddep_launch();
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c = (blockIdx.x * 32 + tx) * VEC;
  const long long r0 = static_cast<long long>(blockIdx.y) * chunk;
  const long long r1 = r0 + chunk < M ? r0 + chunk : M;
  float acc[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
  if (c < N) {
    // rows in flight: with gelu in bf16 147 us at two (32768 x 4608) and 151 at four, in float32 18.1 and 16.7 (4079 x 1536)
    constexpr int U = kFast ? 2 : 4;
    for (long long r = r0 + ty; r < r1; r += 8 * U) {
      Piece<T, VEC> g[U], p[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (r + 8 * u < r1) {
          g[u].ld(dy + (r + 8 * u) * ld_dy + c);
          if (ACT != POM_ACT_NONE) p[u].ld(z + (r + 8 * u) * N + c);
        }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (r + 8 * u < r1) {
          float v[VEC];
          if constexpr (ACT == POM_ACT_NONE) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = g[u].get(e);
          } else if constexpr (VEC == 1) {
            v[0] = g[u].get(0) * linear_slope2<kFast>(ACT, F2(p[u].get(0), 0.f)).v.x;
          } else {
#pragma unroll
            for (int e = 0; e < VEC; e += 2) {
              const F2 s = linear_slope2<kFast>(ACT, F2(p[u].get(e), p[u].get(e + 1)));
              const F2 d = mul2(s, F2(g[u].get(e), g[u].get(e + 1)));
              v[e] = d.v.x, v[e + 1] = d.v.y;
            }
          }
#pragma unroll
          for (int e = 0; e < VEC; ++e) acc[e] += v[e];
          if (ACT != POM_ACT_NONE) {
            g[u].set(v);
            g[u].st(dz + (r + 8 * u) * N + c);
          }
        }
    }
  }
  if (!partial) return;
#pragma unroll
  for (int e = 0; e < VEC; ++e) sm[ty][tx * VEC + e] = acc[e];
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * VEC; i += 256) {
    const int col = blockIdx.x * 32 * VEC + i;
    if (col >= N) continue;
    float s = 0.f;
#pragma unroll
    for (int q = 0; q < 8; ++q) s += sm[q][i];
    partial[static_cast<long long>(blockIdx.y) * N + col] = s;
  }
}

int launched(cudaError_t e) {
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return POM_ERR_CUDA;
  }
  count_launch();
  return POM_OK;
}

FewDev few_dev(const pom_linear_args* a) {
  FewDev d;
  d.x = a->x, d.w = a->w, d.bias = a->bias, d.residual = a->residual;
  d.y = a->y, d.z = a->z;
  d.ldx = a->ldx, d.ldw = a->ldw, d.ldr = a->ldr, d.ldy = a->ldy;
  d.M = static_cast<int>(a->M < INT32_MAX ? a->M : INT32_MAX), d.N = static_cast<int>(a->N), d.K = static_cast<int>(a->K);
  d.act = a->act, d.bias_f32 = a->bias_dtype == POM_F32;
  d.has_bias = a->bias != nullptr, d.has_residual = a->residual != nullptr;
  return d;
}

// An absent bias or residual points at `there`, whose first value has the type `dtype`: a load that the compiler makes ahead of
// its condition finds memory.
FewDev readable(FewDev d, const void* there, int dtype) {
  if (!d.has_bias) d.bias = there, d.bias_f32 = dtype == POM_F32;
  if (!d.has_residual) d.residual = there, d.ldr = 0;
  return d;
}

int check_linear(const pom_linear_args* a) {
  if (!a) return POM_ERR_NULL;
  if (a->M <= 0 || a->N <= 0 || a->K <= 0) return POM_ERR_BAD_SHAPE;
  if (a->M > INT32_MAX || a->N > INT32_MAX || a->K > INT32_MAX) return POM_ERR_TOO_LARGE;
  if (a->dtype != POM_BF16 && a->dtype != POM_F32) return POM_ERR_UNSUPPORTED;
  if (a->bias_dtype != POM_BF16 && a->bias_dtype != POM_F32) return POM_ERR_UNSUPPORTED;
  if (a->act < POM_ACT_NONE || a->act > POM_ACT_RELU) return POM_ERR_UNSUPPORTED;
  return POM_OK;
}

// bf16, this kernel and the tensor cores, weight in HBM (in the L2), us: 1152 -> 4608 at 32 rows 10.2 (6.0) and 14.3 (8.6);
// 1024 -> 1024 at 32 rows 8.2 (3.7) and 12.3 (7.6); 2048 -> 512 12.3 (5.2) and 12.3 (7.8).  Long sums with two tiles of rows wait
// for one trip to memory after the other: 4608 -> 1152 at 32 rows 24.6 (11.4) and 14.3 (10.1), 8192 -> 2048 41.0 (20.6) and 20.5
// (15.5); at 16 rows 12.3 (6.0) and 14.3 (10.1), 20.5 (9.7) and 20.5 (15.5).
constexpr int kFewRowsF32 = 16;

template <int MT>
int launch_few_bf16(const FewDev& d, cudaStream_t st) {
  if (d.M > 16 * MT) return POM_ERR_TOO_LARGE;  // the kernel knows no more rows than its tiles hold
  // two column tiles per block once that still gives every SM a block: x is read half as often
  if (d.N >= 16 * sm_count())
    return launched(launch_pdl(linear_few_bf16_kernel<MT, 2>, dim3(static_cast<unsigned>(ceil_div(d.N, 16))), dim3(32 * kFewWarps), 0, st, d));
  return launched(launch_pdl(linear_few_bf16_kernel<MT, 1>, dim3(static_cast<unsigned>(ceil_div(d.N, 8))), dim3(32 * kFewWarps), 0, st, d));
}

template <int MR>
int launch_few_f32(const FewDev& d, cudaStream_t st) {
  if (d.M > MR) return POM_ERR_TOO_LARGE;
  return launched(launch_pdl(linear_few_f32_kernel<MR>, dim3(static_cast<unsigned>(ceil_div(d.N, 8))), dim3(32 * kFewWarps), 0, st, d));
}

// Row chunks of linear_dz_kernel, at least 32 rows each: one wave of the blocks that an SM holds.  Sums alone, five blocks per
// SM, 32768 x 1152 with the sum of the chunks and from HBM: 28 us (three 34, eight 32).  With dz to write, four: 32768 x 4608
// 154 us, 8192 x 4096 43 (three 168; five 184 and 51; six 171 and 49; eight 155 and 45).
int dz_chunk(int64_t M, int64_t N, int vec, bool sums_only) {
  const int64_t cols = ceil_div(N, 32 * vec), blocks = (sums_only ? 5ll : 4ll) * sm_count();
  const int64_t want = blocks / cols > 0 ? blocks / cols : 1;
  int64_t rows = ceil_div(ceil_div(M, want), 32) * 32;
  if (ceil_div(M, rows) > 65535) rows = ceil_div(ceil_div(M, 65535), 32) * 32;
  return static_cast<int>(rows);
}

uint64_t up256(uint64_t v) { return (v + 255) / 256 * 256; }

// Bytes of the slabs of a bf16 product with (M, N) outputs; 0: it is not cut.
uint64_t slab_bytes(int slabs, int64_t M, int64_t N) {
  return slabs > 1 ? up256(static_cast<uint64_t>(slabs) * M * N * 4) : 0;
}

bool few_rows(const pom_linear_args* a) {
  const int per = a->dtype == POM_BF16 ? 8 : 4;
  return a->M <= (a->dtype == POM_BF16 ? POM_LINEAR_FEW_ROWS(a->K) : kFewRowsF32) && a->K % per == 0 && a->ldx % per == 0 &&
         a->ldw % per == 0 && aligned16(a->x) && aligned16(a->w);
}

// A float32 product on the tensor cores: three bf16 planes of each operand and the partial sums of a cut product, one after
// the other in a workspace.  total 0: on the FMA kernel.
struct F32Plan {
  uint64_t b, scratch, total;
};

constexpr int64_t kF32Rows = 65535ll * 64;  // rows of one float32 product (a grid dimension of the FMA kernel)

// A holds a_rows x a_cols values as it is stored, B b_rows x b_cols.
F32Plan f32_plan(const pom_linear_args* a, int64_t M, int64_t N, int64_t K, int out_mode, int64_t a_rows, int64_t a_cols,
                 int64_t b_rows, int64_t b_cols) {
  F32Plan p{};
  // Short sums run on the FMA kernel (see f32_planes_pay of the Python layer), and so do small products with sums of up to
  // 512 terms: one launch instead of three, which is what such a call waits for (500 x 300 -> 700 in training 139 us
  // against 174), while a longer chain would lose digits that a blocked sum keeps.
  if (a->fma || M > kF32Rows || K < 128 || (K <= 512 && static_cast<double>(M) * static_cast<double>(N) * static_cast<double>(K) < 0x1p27)) return p;
  p.b = up256(pom_f32_planes_bytes(a_rows, a_cols));
  p.scratch = p.b + up256(pom_f32_planes_bytes(b_rows, b_cols));
  p.total = p.scratch + up256(pom_gemm_f32_planes_scratch(M, N, K, out_mode));
  return p;
}

int f32_product(const pom_gemm_args& g, const F32Plan& p, char* ws, int a_ready, int* status, cudaStream_t st) {
  if (!p.total) {
    pom_gemm_args part = g;
    for (int64_t r = 0; r < g.M; r += kF32Rows) {  // more rows than one launch takes (K-major A: the rows of dx and y)
      part.M = g.M - r < kF32Rows || g.a_mn_major ? g.M - r : kF32Rows;
      part.A = static_cast<const float*>(g.A) + r * g.lda;
      part.C = static_cast<float*>(g.C) + r * g.ldc;
      const int rc = pom_gemm_f32(&part, st);
      if (rc || g.a_mn_major) return rc;
    }
    return POM_OK;
  }
  return pom_gemm_f32_planes(&g, ws, a_ready, ws + p.b, 0, ws + p.scratch, status, st);
}

struct BwdPlan {
  int vec, chunk, chunks, dw_slabs;
  uint64_t dz, partial, slab, total;  // byte offsets into the workspace; float32: the planes at `slab`
  F32Plan dw32, dx32;                 // A = dz in both: its planes are made once
};

BwdPlan bwd_plan(const pom_linear_args* a) {
  BwdPlan p{};
  const int per = a->dtype == POM_BF16 ? 8 : 4;
  p.vec = a->N % per || a->ld_dy % per || !aligned16(a->dy) || !aligned16(a->z) ? 1 : per;  // bf16: refused unless wide
  p.chunk = dz_chunk(a->M, a->N, p.vec, a->act == POM_ACT_NONE);
  p.chunks = static_cast<int>(ceil_div(a->M, p.chunk));
  const bool bf16 = a->dtype == POM_BF16;
  p.dw_slabs = bf16 && a->dw ? gemm_bf16_slabs(a->N, a->K, a->M, true, true) : 1;
  uint64_t at = 0;
  p.dz = at;
  if (a->act != POM_ACT_NONE) at = up256(at + static_cast<uint64_t>(a->M) * a->N * (bf16 ? 2 : 4));
  p.partial = at;
  if (a->dbias) at = up256(at + static_cast<uint64_t>(p.chunks) * a->N * 4);
  p.slab = at;
  p.total = at + slab_bytes(p.dw_slabs, a->N, a->K);
  if (!bf16) {
    // dw sums over the rows and has few output tiles: it is accumulated, since only that may be cut along its sum
    if (a->dw) p.dw32 = f32_plan(a, a->N, a->K, a->M, POM_OUT_F32_ACCUM, a->M, a->N, a->M, a->K);
    if (a->dx) p.dx32 = f32_plan(a, a->M, a->K, a->N, POM_OUT_F32, a->M, a->N, a->N, a->K);
    p.total = at + (p.dw32.total > p.dx32.total ? p.dw32.total : p.dx32.total);
  }
  return p;
}

// d.y = act(sum of slabs + bias) + residual in bf16 (T) or fp32.
template <class T, int VEC>
int launch_epilogue(const FewDev& few, const float* z, int64_t ldz, int slabs, int64_t M, cudaStream_t st) {
  const FewDev d = readable(few, z, POM_F32);
  const int64_t want = ceil_div(M * (d.N / VEC), 256), cap = 16ll * sm_count();
  const dim3 grid(static_cast<unsigned>(want < cap ? want : cap));
  const long long ld = ldz, rows = M;
  return launched(launch_pdl(linear_epilogue_kernel<T, VEC>, grid, dim3(256), 0, st, d, z, ld, slabs, rows));
}

// g, whose output is bf16 and contiguous, whole or as slabs and their sum.
int product(pom_gemm_args g, int slabs, float* slab, int* status, cudaStream_t st) {
  void* out = g.C;
  if (slabs > 1) g.C = slab, g.out_mode = POM_OUT_F32;
  const int rc = gemm_bf16_slabs(&g, slabs, status, st);
  if (rc || slabs <= 1) return rc;
  FewDev d{};
  d.y = out, d.ldy = g.N, d.N = static_cast<int>(g.N);
  return launch_epilogue<__nv_bfloat16, 4>(d, slab, g.N, slabs, g.M, st);  // the engine takes widths of multiples of 8
}

template <class T, int VEC>
int launch_dz(const pom_linear_args* a, const BwdPlan& p, void* dz, float* partial, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(ceil_div(a->N, 32 * VEC)), static_cast<unsigned>(p.chunks));
  const long long M = a->M, ld = a->ld_dy;
  const int N = static_cast<int>(a->N);
#define POM_DZ(ACT)                                                                                                     \
  case ACT:                                                                                                             \
    return launched(launch_pdl(linear_dz_kernel<T, VEC, ACT>, grid, dim3(256), 0, st, static_cast<const T*>(a->dy), ld, \
                               static_cast<const T*>(a->z), static_cast<T*>(dz), partial, M, N, p.chunk));
  switch (a->act) {
    POM_DZ(POM_ACT_NONE)
    POM_DZ(POM_ACT_GELU)
    POM_DZ(POM_ACT_GELU_TANH)
    POM_DZ(POM_ACT_SILU)
    POM_DZ(POM_ACT_RELU)
  }
#undef POM_DZ
  return POM_ERR_UNSUPPORTED;
}

// dz (with an activation) and dbias.
int dz_and_bias(const pom_linear_args* a, const BwdPlan& p, void* dz, cudaStream_t st) {
  if (a->act == POM_ACT_NONE && !a->dbias) return POM_OK;
  float* partial = a->dbias ? reinterpret_cast<float*>(static_cast<char*>(a->workspace) + p.partial) : nullptr;
  const int N = static_cast<int>(a->N);
  const int rc = a->dtype == POM_BF16
                     ? launch_dz<__nv_bfloat16, 8>(a, p, dz, partial, st)
                     : (p.vec == 4 ? launch_dz<float, 4>(a, p, dz, partial, st) : launch_dz<float, 1>(a, p, dz, partial, st));
  if (rc || !partial) return rc;
  return sum_rows(partial, p.chunks, N, N, a->bias_dtype, a->dbias, nullptr, st);
}

}  // namespace

extern "C" {

int pom_linear_fwd(const pom_linear_args* a, int* status, void* stream) {
  int rc = check_linear(a);
  if (rc) return rc;
  if (!a->x || !a->w || !a->y) return POM_ERR_NULL;
  if (a->ldx < a->K || a->ldw < a->K || a->ldy < a->N || (a->residual && a->ldr < a->N)) return POM_ERR_BAD_STRIDE;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (few_rows(a)) {
    const FewDev d = readable(few_dev(a), a->x, a->dtype);
    if (a->dtype == POM_BF16) {
      return a->M <= 16 ? launch_few_bf16<1>(d, st) : launch_few_bf16<2>(d, st);
    }
    if (a->M == 1) return launch_few_f32<1>(d, st);
    if (a->M <= 4) return launch_few_f32<4>(d, st);
    if (a->M <= 8) return launch_few_f32<8>(d, st);
    return launch_few_f32<16>(d, st);
  }
  if (a->dtype == POM_F32) {
    const F32Plan p = f32_plan(a, a->M, a->N, a->K, POM_OUT_F32, a->M, a->K, a->N, a->K);
    if (p.total && !a->workspace) return POM_ERR_NULL;
    if (!aligned16(a->workspace)) return POM_ERR_BAD_ALIGN;
    pom_gemm_args g{};
    g.A = a->x, g.Bm = a->w, g.C = a->y;
    g.M = a->M, g.N = a->N, g.K = a->K;
    g.lda = a->ldx, g.ldb = a->ldw, g.ldc = a->ldy;
    g.batches = 1, g.split_k = 1, g.alpha = 1.f, g.out_mode = POM_OUT_F32;
    if ((rc = f32_product(g, p, static_cast<char*>(a->workspace), 0, status, st))) return rc;
    if (!a->bias && !a->residual && !a->z && a->act == POM_ACT_NONE) return POM_OK;
    const bool wide = a->N % 4 == 0 && a->ldy % 4 == 0 && aligned16(a->y) && aligned16(a->z) &&
                      (!a->residual || (a->ldr % 4 == 0 && aligned16(a->residual)));
    const float* sums = static_cast<const float*>(a->y);
    return wide ? launch_epilogue<float, 4>(few_dev(a), sums, a->ldy, 1, a->M, st)
                : launch_epilogue<float, 1>(few_dev(a), sums, a->ldy, 1, a->M, st);
  }
  Operands o{a->x, a->w, a->M, a->N, a->K, a->ldx, a->ldw, 1, false, false};
  if ((rc = check_operands(o))) return rc;
  const ClusterPlan cp = pick_cluster(a->M, a->N, a->K);
  if (cp.size > 1) {
    if (a->N % 8 || a->ldy % 8 || (a->residual && a->ldr % 8)) return POM_ERR_BAD_STRIDE;
    if (!aligned16(a->y) || !aligned16(a->z) || !aligned16(a->residual)) return POM_ERR_BAD_ALIGN;
    ClusterDev d{};
    d.bias = a->bias, d.has_bias = a->bias != nullptr, d.bias_f32 = a->bias_dtype == POM_F32, d.act = a->act;
    d.residual = static_cast<const __nv_bfloat16*>(a->residual), d.has_residual = a->residual != nullptr, d.ldr = a->ldr;
    d.y = static_cast<__nv_bfloat16*>(a->y), d.ldy = a->ldy;
    d.z = static_cast<__nv_bfloat16*>(a->z);
    return cluster_product(o, cp, d, status, st);
  }
  EpiMaps maps{};
  if (a->z && (rc = make_io_map(&maps.out0, a->z, a->N, a->M, 1, a->N))) return rc;
  if ((rc = make_io_map(&maps.out1, a->y, a->N, a->M, 1, a->ldy))) return rc;
  if (a->residual) {
    if ((rc = make_io_map(&maps.in0, a->residual, a->N, a->M, 1, a->ldr))) return rc;
    const EpiLinear<true>::Params ep{a->bias ? a->bias : a->x, a->bias != nullptr, a->bias_dtype == POM_F32, a->act, a->z != nullptr};
    return run_plan<false, false, EpiLinear<true>>(pick_plan(o, true), o, 1, maps, ep, status, st);
  }
  const EpiLinear<false>::Params ep{a->bias ? a->bias : a->x, a->bias != nullptr, a->bias_dtype == POM_F32, a->act, a->z != nullptr};
  return run_plan<false, false, EpiLinear<false>>(pick_plan(o, true), o, 1, maps, ep, status, st);
}

uint64_t pom_linear_fwd_workspace(const pom_linear_args* a) {
  if (check_linear(a) || a->dtype != POM_F32 || few_rows(a)) return 0;
  return f32_plan(a, a->M, a->N, a->K, POM_OUT_F32, a->M, a->K, a->N, a->K).total;
}

uint64_t pom_linear_bwd_workspace(const pom_linear_args* a) { return check_linear(a) ? 0 : bwd_plan(a).total; }

int pom_linear_bwd(const pom_linear_args* a, int* status, void* stream) {
  int rc = check_linear(a);
  if (rc) return rc;
  if (!a->dy || (a->act != POM_ACT_NONE && !a->z) || (a->dw && !a->x) || (a->dx && !a->w)) return POM_ERR_NULL;
  if (a->ld_dy < a->N || (a->dx && a->ldw < a->K) || (a->dw && a->ldx < a->K)) return POM_ERR_BAD_STRIDE;
  const BwdPlan p = bwd_plan(a);
  if (p.total && !a->workspace) return POM_ERR_NULL;
  if (!aligned16(a->workspace)) return POM_ERR_BAD_ALIGN;
  if (a->dtype == POM_BF16) {
    if (p.vec == 1 && (a->N % 8 || a->ld_dy % 8)) return POM_ERR_BAD_STRIDE;
    if (p.vec == 1 || !aligned16(a->dw) || !aligned16(a->dx)) return POM_ERR_BAD_ALIGN;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(a->workspace);
  if ((rc = dz_and_bias(a, p, ws + p.dz, st))) return rc;
  const bool own = a->act != POM_ACT_NONE;
  const void* dz = own ? ws + p.dz : a->dy;
  const int64_t ld_dz = own ? a->N : a->ld_dy;
  pom_gemm_args g{};
  g.batches = 1, g.split_k = 1, g.alpha = 1.f;
  const bool f32 = a->dtype == POM_F32;
  if (a->dw) {
    g.A = dz, g.Bm = a->x, g.C = a->dw;
    g.M = a->N, g.N = a->K, g.K = a->M;
    g.lda = ld_dz, g.ldb = a->ldx, g.ldc = a->K;
    g.a_mn_major = g.b_mn_major = 1;
    if (f32) {
      g.out_mode = p.dw32.total ? POM_OUT_F32_ACCUM : POM_OUT_F32;
      if (p.dw32.total && (rc = pom_fill_zero(a->dw, a->N * a->K * 4, st))) return rc;
      rc = f32_product(g, p.dw32, ws + p.slab, 0, status, st);
    } else {
      g.out_mode = POM_OUT_BF16;
      rc = product(g, p.dw_slabs, reinterpret_cast<float*>(ws + p.slab), status, st);
    }
    if (rc) return rc;
  }
  if (a->dx) {
    g.A = dz, g.Bm = a->w, g.C = a->dx;
    g.M = a->M, g.N = a->K, g.K = a->N;
    g.lda = ld_dz, g.ldb = a->ldw, g.ldc = a->K;
    g.a_mn_major = 0, g.b_mn_major = 1;
    g.out_mode = f32 ? POM_OUT_F32 : POM_OUT_BF16;
    const ClusterPlan cp = f32 ? ClusterPlan{128, 1} : pick_cluster(a->M, a->K, a->N);
    if (f32) {
      rc = f32_product(g, p.dx32, ws + p.slab, p.dw32.total != 0, status, st);
    } else if (cp.size > 1) {
      Operands o{dz, a->w, a->M, a->K, a->N, ld_dz, a->ldw, 1, false, true};
      ClusterDev d{};
      d.y = static_cast<__nv_bfloat16*>(a->dx), d.ldy = a->K;
      rc = cluster_product(o, cp, d, status, st);
    } else {
      rc = pom_gemm_bf16(&g, status, st);
    }
    if (rc) return rc;
  }
  return check_launch();
}
}  // extern "C"
