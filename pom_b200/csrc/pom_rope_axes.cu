// Rotary positions of one to four axes (time, height, width, ...).
//
// The channels of x (B, N, H, D) are cut into one section per axis, 2 s_a channels wide and in the order of the axes;
// channel k of a section is paired with channel k + s_a, and the pair is turned by the angle whose cosine and sine stand
// in row position_a, column k of the axis' table:
//     y[k] = x[k] cos - x[k + s] sin        y[k + s] = x[k] sin + x[k + s] cos
// The transpose (the backward pass) turns the other way.  Channels behind the last section are copied.
//
// A thread owns VEC pairs (16 bytes on either side of the pairing where alignment allows) of one head and walks a run of
// tokens, the next one's loads in flight: where its channels lie is found once, and a step of the walk is two loads of x, one
// position and the table row that it names.  Bound by HBM: 302 MB in 56 to 59 us (5.1 to 5.3 TB/s; 32768 tokens of 2304 bf16
// channels).  Runs of 16 tokens take 64 to 70 us there; pieces without a walk 57, but 19.4 instead of 15.8 with 16 heads of 72.
#include <limits.h>
#include <initializer_list>
#include "rows.cuh"

using namespace pomk;
using namespace pomh;

namespace {

constexpr int kMaxAxes = POM_ROPE_MAX_AXES;
constexpr int kThreads = 256, kPerSm = 8, kRun = 8;

struct AxesDev {
  const void* x;
  void* y;
  const long long* pos;  // (N, axes), or (B, N, axes)
  const float* cos[kMaxAxes];
  const float* sin[kMaxAxes];
  int len[kMaxAxes], pairs[kMaxAxes];
  long long xs_b, xs_n, xs_h;  // strides of x; y is contiguous
  long long B, N;
  int H, D, axes, units, pair_units, run;
  int pos_per_sample;
  float sign;
};

template <class T, int VEC>
__global__ void __launch_bounds__(kThreads) rope_axes_kernel(const AxesDev a) {
  griddep_wait();
  griddep_launch();
  const int hu = blockIdx.y * blockDim.x + threadIdx.x;
  if (hu >= a.H * a.units) return;
  const int h = hu / a.units;
  int u = hu - h * a.units;
  // where this thread's channels lie: section `axis`, pairs k .. k + VEC of it, first channel lo + k; axis < 0: copied
  int axis = -1, lo = 0, s = 0, k = a.D - (a.units - u) * VEC;
  const float *ct = nullptr, *st = nullptr;
  int len = 0;
  if (u < a.pair_units) {
    axis = 0;
    while (u * VEC >= a.pairs[axis]) u -= a.pairs[axis] / VEC, lo += 2 * a.pairs[axis], ++axis;
    s = a.pairs[axis], k = u * VEC, len = a.len[axis];
    ct = a.cos[axis] + k, st = a.sin[axis] + k;
  }
  const T* __restrict__ x = static_cast<const T*>(a.x) + h * a.xs_h + lo + k;
  T* __restrict__ y = static_cast<T*>(a.y) + h * static_cast<long long>(a.D) + lo + k;
  const long long* __restrict__ pos = a.pos + axis;
  const long long y_tok = static_cast<long long>(a.H) * a.D, total = a.B * a.N;
  const long long tok0 = static_cast<long long>(blockIdx.x) * a.run * blockDim.y + threadIdx.y;
  const long long stop = tok0 - threadIdx.y + static_cast<long long>(a.run) * blockDim.y, end = stop < total ? stop : total;
  // what a token needs from global memory, one token ahead of its turn
  Piece<T, VEC> n1, n2;
  long long np = 0;
  auto fetch = [&](long long tok) {
    if (tok >= end) return;
    const long long b = total <= 0x7fffffff ? static_cast<unsigned>(tok) / static_cast<unsigned>(a.N) : tok / a.N;
    const long long n = tok - b * a.N;
    const T* xr = x + b * a.xs_b + n * a.xs_n;
    n1.ld(xr);
    if (axis >= 0) {
      n2.ld(xr + s);
      np = __ldg(pos + (a.pos_per_sample ? tok : n) * a.axes);
    }
  };
  fetch(tok0);
  for (long long tok = tok0; tok < end; tok += blockDim.y) {
    Piece<T, VEC> p1 = n1, p2 = n2;
    const long long p = np;
    fetch(tok + blockDim.y);
    T* yr = y + tok * y_tok;
    if (axis < 0) {
      p1.st(yr);
      continue;
    }
    float cs[VEC], sn[VEC];
    if (p >= 0 && p < len) {
      constexpr int F = VEC < 4 ? VEC : 4;
#pragma unroll
      for (int e = 0; e < VEC; e += F) {
        Piece<float, F> pc, ps;
        pc.ld(ct + p * s + e), ps.ld(st + p * s + e);
#pragma unroll
        for (int f = 0; f < F; ++f) cs[e + f] = pc.get(f), sn[e + f] = a.sign * ps.get(f);
      }
    } else {  // no such row: not a number, and never a read outside the table
#pragma unroll
      for (int e = 0; e < VEC; ++e) cs[e] = sn[e] = __int_as_float(0x7fc00000);
    }
    float v1[VEC], v2[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float x1 = p1.get(e), x2 = p2.get(e);
      v1[e] = x1 * cs[e] - x2 * sn[e];
      v2[e] = x1 * sn[e] + x2 * cs[e];
    }
    p1.set(v1), p2.set(v2);
    p1.st(yr);
    p2.st(yr + s);
  }
}

// Smallest and largest position per axis of the block's rows, written side by side to the host's memory.
__global__ void __launch_bounds__(1024) pos_range_kernel(const long long* __restrict__ pos, long long rows, int axes,
                                                         long long* host_info) {
  __shared__ long long sm[2 * kMaxAxes][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long hi[kMaxAxes], lo[kMaxAxes];
#pragma unroll
  for (int c = 0; c < kMaxAxes; ++c) hi[c] = LLONG_MIN, lo[c] = LLONG_MAX;
#pragma unroll 4
  for (long long i = blockIdx.x * 1024ll + threadIdx.x; i < rows; i += gridDim.x * 1024ll)
#pragma unroll
    for (int c = 0; c < kMaxAxes; ++c)
      if (c < axes) {
        const long long p = __ldg(pos + i * axes + c);
        hi[c] = p > hi[c] ? p : hi[c];
        lo[c] = p < lo[c] ? p : lo[c];
      }
#pragma unroll
  for (int c = 0; c < kMaxAxes; ++c) {
    for (int o = 16; o; o >>= 1) {
      const long long h = __shfl_xor_sync(0xffffffffu, hi[c], o), l = __shfl_xor_sync(0xffffffffu, lo[c], o);
      hi[c] = h > hi[c] ? h : hi[c];
      lo[c] = l < lo[c] ? l : lo[c];
    }
    if (lane == 0) sm[2 * c][warp] = lo[c], sm[2 * c + 1][warp] = hi[c];
  }
  __syncthreads();
  if (warp < 2 * axes) {  // warp w finishes value w
    long long v = sm[warp][lane];
    for (int o = 16; o; o >>= 1) {
      const long long t = __shfl_xor_sync(0xffffffffu, v, o);
      v = (warp & 1) ? (t > v ? t : v) : (t < v ? t : v);
    }
    if (lane == 0) {
      host_info[blockIdx.x * 2 * axes + warp] = v;
      __threadfence_system();  // now, not with the end of whatever follows
    }
  }
}

// Pairs per thread: 16 bytes of x where every section, stride and address allows it, else 8, 4 bytes, else one value.
int axes_vec(const pom_rope_axes_args* a, int wide) {
  for (int v : {wide, 4, 2}) {
    bool ok = a->D % v == 0 && a->xs_b % v == 0 && a->xs_n % v == 0 && a->xs_h % v == 0;
    const uintptr_t xm = static_cast<uintptr_t>(v) * (a->dtype == POM_BF16 ? 2 : 4) - 1;
    const uintptr_t fm = (v < 4 ? v : 4) * 4 - 1;
    ok = ok && !((reinterpret_cast<uintptr_t>(a->x) | reinterpret_cast<uintptr_t>(a->y)) & xm);
    for (int i = 0; i < a->axes; ++i)
      ok = ok && a->pairs[i] % v == 0 &&
           !((reinterpret_cast<uintptr_t>(a->cos[i]) | reinterpret_cast<uintptr_t>(a->sin[i])) & fm);
    if (ok) return v;
  }
  return 1;
}

}  // namespace

extern "C" {

int pom_rope_axes(const pom_rope_axes_args* a, void* stream) {
  if (!a || !a->x || !a->y || !a->pos) return POM_ERR_NULL;
  if (a->axes < 1 || a->axes > kMaxAxes) return POM_ERR_UNSUPPORTED;
  if (a->dtype != POM_BF16 && a->dtype != POM_F32) return POM_ERR_UNSUPPORTED;
  if (a->B <= 0 || a->N <= 0 || a->H <= 0 || a->D <= 0) return POM_ERR_BAD_SHAPE;
  if (a->xs_b < 0 || a->xs_n < 0 || a->xs_h < 0) return POM_ERR_BAD_STRIDE;
  AxesDev d;
  long long total_pairs = 0;
  for (int i = 0; i < kMaxAxes; ++i) {
    d.cos[i] = a->cos[i], d.sin[i] = a->sin[i], d.len[i] = a->len[i], d.pairs[i] = a->pairs[i];
    if (i >= a->axes) continue;
    if (!a->cos[i] || !a->sin[i]) return POM_ERR_NULL;
    if (a->len[i] <= 0 || a->pairs[i] <= 0) return POM_ERR_BAD_SHAPE;
    total_pairs += a->pairs[i];
  }
  if (2 * total_pairs > a->D) return POM_ERR_BAD_SHAPE;
  const int vec = axes_vec(a, a->dtype == POM_BF16 ? 8 : 4);
  d.x = a->x, d.y = a->y, d.pos = reinterpret_cast<const long long*>(a->pos);
  d.xs_b = a->xs_b, d.xs_n = a->xs_n, d.xs_h = a->xs_h;
  d.B = a->B, d.N = a->N, d.H = a->H, d.D = a->D, d.axes = a->axes;
  d.pair_units = static_cast<int>(total_pairs / vec);
  d.units = d.pair_units + static_cast<int>((a->D - 2 * total_pairs) / vec);
  d.pos_per_sample = a->pos_per_sample;
  d.sign = a->transpose ? -1.f : 1.f;
  // blockDim = (pieces of a token: heads x units, tokens); blockIdx = (token lanes, pieces)
  const int64_t per_tok = static_cast<int64_t>(a->H) * d.units, tokens = a->B * a->N;
  if (per_tok > 65535ll * 256) return POM_ERR_TOO_LARGE;
  const int64_t bx = per_tok < 256 ? per_tok : 256, by = kThreads / bx, pieces = ceil_div(per_tok, bx);
  int64_t run = tokens * pieces / (kPerSm * sm_count() * by);
  run = run < 1 ? 1 : run > kRun ? kRun : run;
  if (ceil_div(tokens, run * by) > INT32_MAX) return POM_ERR_TOO_LARGE;
  d.run = static_cast<int>(run);
  const dim3 grid(static_cast<unsigned>(ceil_div(tokens, run * by)), static_cast<unsigned>(pieces));
  const dim3 block(static_cast<unsigned>(bx), static_cast<unsigned>(by));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
#define POM_AXES(T, V) e = launch_pdl(rope_axes_kernel<T, V>, grid, block, 0, st, d)
  if (a->dtype == POM_BF16) {
    if (vec == 8) POM_AXES(__nv_bfloat16, 8);
    else if (vec == 4) POM_AXES(__nv_bfloat16, 4);
    else if (vec == 2) POM_AXES(__nv_bfloat16, 2);
    else POM_AXES(__nv_bfloat16, 1);
  } else {
    if (vec == 4) POM_AXES(float, 4);
    else if (vec == 2) POM_AXES(float, 2);
    else POM_AXES(float, 1);
  }
#undef POM_AXES
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return POM_ERR_CUDA;
  }
  count_launch();
  return check_launch();
}

int32_t pom_pos_range_blocks(int64_t rows) {
  const int64_t want = ceil_div(rows, 16384);  // the host looks at every block's values, so few blocks for few rows
  return static_cast<int32_t>(want < 1 ? 1 : want < POM_POS_RANGE_BLOCKS ? want : POM_POS_RANGE_BLOCKS);
}

int pom_pos_range(const int64_t* pos, int64_t rows, int32_t axes, int64_t* host_info, void* stream) {
  if (!pos || !host_info) return POM_ERR_NULL;
  if (rows <= 0 || axes < 1 || axes > kMaxAxes) return POM_ERR_BAD_SHAPE;
  pos_range_kernel<<<static_cast<unsigned>(pom_pos_range_blocks(rows)), 1024, 0, static_cast<cudaStream_t>(stream)>>>(
      reinterpret_cast<const long long*>(pos), rows, axes, reinterpret_cast<long long*>(host_info));
  count_launch();
  return check_launch();
}
}  // extern "C"
