// Layer norm over the last dimension, forward and backward.
//
//   m = mean(x), r = (mean((x - m)^2) + eps)^(-1/2), xh = (x - m) r        y = xh w + b
//   dx = r (h - mean(h) - xh mean(h xh)),  h = g w        dw = sum_rows g xh        db = sum_rows g
//
// Both directions read every row once: a row is held in the registers of TPR threads (NV pieces of VEC values each), so
// the variance is taken around the mean that was just found (no difference of two large sums) and the backward sums and
// dx come from the same registers.  All sums are fp32.  The gradients of w and b are summed over the rows a thread walks
// in registers, over the warps of a block in a fixed order, and written as one row per block; a second kernel adds
// those rows in a fixed order: the same bits on every run.
#include <initializer_list>
#include "f32x2.cuh"
#include "rows.cuh"

using namespace pomk;
using namespace pomh;

namespace {

struct NormDev {
  const void* x;
  const void* w;  // without a scale (has_w 0): x, so that nothing is ever read at an address that does not exist
  const void* b;  // without a shift (has_b 0): w
  void* y;
  float2* stats;  // (mean, r) per row, or null (forward)
  const void* dy;
  void* dx;        // or null
  float* partial;  // (blocks, 2, D) or null
  long long M, ldx, ldy, ld_dy, ld_dx;
  int D;
  int has_w, has_b;
  float eps;
};

// Sum over the TPR threads of a row, the same value (and bits) in all of them.  `slot` alternates between two halves of
// `sm`, so one barrier per sum is enough.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* sm, int slot) {
  v = warp_sum(v);
  if constexpr (TPR == 32) return v;
  constexpr int kWarps = TPR / 32;
  if ((threadIdx.x & 31) == 0) sm[slot * kWarps + (threadIdx.x >> 5)] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) s += sm[slot * kWarps + i];
  return s;
}

template <int TPR>
__device__ __forceinline__ float2 row_sum2(float a, float b, float2* sm, int slot) {
  a = warp_sum(a), b = warp_sum(b);
  if constexpr (TPR == 32) return make_float2(a, b);
  constexpr int kWarps = TPR / 32;
  if ((threadIdx.x & 31) == 0) sm[slot * kWarps + (threadIdx.x >> 5)] = make_float2(a, b);
  __syncthreads();
  float2 s = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < kWarps; ++i) s.x += sm[slot * kWarps + i].x, s.y += sm[slot * kWarps + i].y;
  return s;
}

// TPR == 32: a warp per row, several rows per block; else a block per row.  Bound by HBM: 32768 x 1152 bf16 takes 30 us (151 MB,
// 5.0 TB/s; 1152 channels leave a tenth of the lanes idle, 1024 channels none: 5.75 TB/s).
template <class T, class W, int VEC, int NV, int TPR>
__global__ void norm_fwd_kernel(const NormDev a) {
  __shared__ float sm[2 * (TPR / 32)];
  griddep_wait();
  griddep_launch();
  const int t = TPR == 32 ? threadIdx.x & 31 : threadIdx.x;
  const int sub = TPR == 32 ? threadIdx.x >> 5 : 0;
  const int rows = TPR == 32 ? blockDim.x >> 5 : 1;
  const float inv_d = 1.f / static_cast<float>(a.D);
  for (long long row = static_cast<long long>(blockIdx.x) * rows + sub; row < a.M; row += static_cast<long long>(gridDim.x) * rows) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    Piece<T, VEC> p[NV];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * VEC;
      if (c < a.D) p[i].ld(x + c);
      else p[i].zero();
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) s += p[i].get(e);
    const float mean = row_sum<TPR>(s, sm, 0) * inv_d;
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((i * TPR + t) * VEC < a.D) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float d = p[i].get(e) - mean;
          q = fmaf(d, d, q);
        }
      }
    const float r = rsqrtf(row_sum<TPR>(q, sm, 1) * inv_d + a.eps);
    if (a.stats && t == 0) a.stats[row] = make_float2(mean, r);
    T* y = static_cast<T*>(a.y) + row * a.ldy;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * VEC;
      if (c < a.D) {
        float o[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) o[e] = (p[i].get(e) - mean) * r;
        if (a.has_w) {
          constexpr int WV = VEC * static_cast<int>(sizeof(W)) <= 16 ? VEC : 16 / static_cast<int>(sizeof(W));
          const W* w = static_cast<const W*>(a.w) + c;
          const W* b = static_cast<const W*>(a.b) + c;
#pragma unroll
          for (int k = 0; k < VEC; k += WV) {
            Piece<W, WV> pw, pb;
            pw.ld(w + k);
            if (a.has_b) pb.ld(b + k);
            else pb.zero();
#pragma unroll
            for (int e = 0; e < WV; ++e) o[k + e] = fmaf(o[k + e], pw.get(e), pb.get(e));
          }
        }
        p[i].set(o);
        p[i].st(y + c);
      }
    }
  }
}

// Rows too wide for the registers of a block: three passes over a row that stays in the caches.
template <class T, class W>
__global__ void __launch_bounds__(512) norm_fwd_wide_kernel(const NormDev a) {
  __shared__ float sm[32];
  griddep_wait();
  griddep_launch();
  const float inv_d = 1.f / static_cast<float>(a.D);
  for (long long row = blockIdx.x; row < a.M; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    T* y = static_cast<T*>(a.y) + row * a.ldy;
    Piece<T, 1> p;
    float s = 0.f, q = 0.f;
    for (int c = threadIdx.x; c < a.D; c += 512) p.ld(x + c), s += p.get(0);
    const float mean = row_sum<512>(s, sm, 0) * inv_d;
    for (int c = threadIdx.x; c < a.D; c += 512) {
      p.ld(x + c);
      const float d = p.get(0) - mean;
      q = fmaf(d, d, q);
    }
    const float r = rsqrtf(row_sum<512>(q, sm, 1) * inv_d + a.eps);
    if (a.stats && threadIdx.x == 0) a.stats[row] = make_float2(mean, r);
    for (int c = threadIdx.x; c < a.D; c += 512) {
      p.ld(x + c);
      float o[1] = {(p.get(0) - mean) * r};
      if (a.has_w) {
        Piece<W, 1> pw, pb;
        pw.ld(static_cast<const W*>(a.w) + c);
        if (a.has_b) pb.ld(static_cast<const W*>(a.b) + c);
        else pb.zero();
        o[0] = fmaf(o[0], pw.get(0), pb.get(0));
      }
      p.set(o);
      p.st(y + c);
    }
  }
}

// Backward, bound by HBM: 32768 x 1152 bf16 takes 51 us (226 MB, 4.4 TB/s); with one row in flight and scalar arithmetic 82.
// The row's pieces a thread will read come through shared memory, kStages - 1 rows ahead, with asynchronous copies: every
// thread copies exactly the 16 bytes that it reads itself, so no barrier stands between copy and use.
__device__ __forceinline__ void copy16(uint4* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// rows in flight per thread group: what fits beside the widest rows' scale (512 threads: 196 KB at two)
template <int TPR>
constexpr int kBwdStages = TPR == 512 ? 2 : 3;

// 16-byte pieces (VEC 8 or 4).  scratch: [w: (NV, TPR, VEC) floats][ring: stage, x or dy, piece, thread]; after the rows,
// with TPR == 32, the first 2 * D floats hold the block's sums.
template <class T, class W, int NV, int TPR>
__global__ void __launch_bounds__(TPR == 32 ? 384 : TPR, TPR == 128 ? 3 : 1) norm_bwd_kernel(const NormDev a) {
  constexpr int VEC = 16 / static_cast<int>(sizeof(T)), P2 = VEC / 2, kStages = kBwdStages<TPR>;
  extern __shared__ uint4 scratch[];
  __shared__ float2 sm[2 * (TPR / 32)];
  const int t = TPR == 32 ? threadIdx.x & 31 : threadIdx.x;
  const int sub = TPR == 32 ? threadIdx.x >> 5 : 0;
  const int rows = TPR == 32 ? blockDim.x >> 5 : 1;
  float* wsm = reinterpret_cast<float*>(scratch);  // piece i of thread t at (i * TPR + t) * VEC: column order
  uint4* ring = scratch + NV * TPR * VEC / 4 + threadIdx.x;
  const int T0 = blockDim.x;
  griddep_wait();
  griddep_launch();
  const float inv_d = 1.f / static_cast<float>(a.D);
  const bool affine = a.has_w;
  for (int c = threadIdx.x; c < NV * TPR * VEC; c += T0) {
    Piece<W, 1> p;
    p.zero();
    if (affine && c < a.D) p.ld(static_cast<const W*>(a.w) + c);
    wsm[c] = affine ? p.get(0) : 1.f;
  }
  const long long step = static_cast<long long>(gridDim.x) * rows;
  const long long first = static_cast<long long>(blockIdx.x) * rows + sub;
  auto fetch = [&](long long row, int stage) {
    if (row < a.M) {
      const T* x = static_cast<const T*>(a.x) + row * a.ldx;
      const T* g = static_cast<const T*>(a.dy) + row * a.ld_dy;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * TPR + t) * VEC;
        if (c < a.D) {
          copy16(ring + ((stage * 2 + 0) * NV + i) * T0, x + c);
          copy16(ring + ((stage * 2 + 1) * NV + i) * T0, g + c);
        }
      }
    }
    copy_commit();
  };
  for (int s = 0; s < kStages - 1; ++s) fetch(first + s * step, s);
  float2 st = first < a.M ? __ldg(a.stats + first) : make_float2(0.f, 0.f);
  F2 dw[NV][P2], db[NV][P2];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < P2; ++e) dw[i][e] = db[i][e] = F2(0.f);
  __syncthreads();
  int slot = 0, stage = 0;
  for (long long row = first; row < a.M; row += step) {
    int ahead = stage + kStages - 1;
    if (ahead >= kStages) ahead -= kStages;
    fetch(row + (kStages - 1) * step, ahead);  // into the stage that the previous row has left
    const float mean = st.x, r = st.y;
    if (row + step < a.M) st = __ldg(a.stats + row + step);
    copy_wait<kStages - 1>();
    const F2 r2(r), off(-mean * r);
    Piece<T, VEC> px[NV], pg[NV];
    F2 s1(0.f), s2(0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * VEC;
      if (c < a.D) {
        px[i].raw = ring[((stage * 2 + 0) * NV + i) * T0];
        pg[i].raw = ring[((stage * 2 + 1) * NV + i) * T0];
#pragma unroll
        for (int e = 0; e < P2; ++e) {
          const F2 g(pg[i].get(2 * e), pg[i].get(2 * e + 1)), x(px[i].get(2 * e), px[i].get(2 * e + 1));
          const F2 xh = fma2(x, r2, off);
          const float2 w = *reinterpret_cast<const float2*>(wsm + c + 2 * e);
          const F2 h = mul2(g, F2(w.x, w.y));
          s1 = add2(s1, h);
          s2 = fma2(h, xh, s2);
          dw[i][e] = fma2(g, xh, dw[i][e]);
          db[i][e] = add2(db[i][e], g);
        }
      }
    }
    if (++stage == kStages) stage = 0;
    if (!a.dx) continue;  // the same for every thread
    const float2 s = row_sum2<TPR>(s1.v.x + s1.v.y, s2.v.x + s2.v.y, sm, slot);
    slot ^= 1;
    // dx = r h - r c1 - xh (r c2)
    const F2 c1(-r * (s.x * inv_d)), c2(-r * (s.y * inv_d));
    T* dx = static_cast<T*>(a.dx) + row * a.ld_dx;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * VEC;
      if (c < a.D) {
        float o[VEC];
#pragma unroll
        for (int e = 0; e < P2; ++e) {
          const F2 g(pg[i].get(2 * e), pg[i].get(2 * e + 1)), x(px[i].get(2 * e), px[i].get(2 * e + 1));
          const F2 xh = fma2(x, r2, off);
          const float2 w = *reinterpret_cast<const float2*>(wsm + c + 2 * e);
          const F2 d = fma2(mul2(g, F2(w.x, w.y)), r2, fma2(xh, c2, c1));
          o[2 * e] = d.v.x, o[2 * e + 1] = d.v.y;
        }
        px[i].set(o);
        px[i].st(dx + c);
      }
    }
  }
  copy_wait<0>();
  if (!a.partial) return;
  float* out = a.partial + static_cast<long long>(blockIdx.x) * 2 * a.D;
  if constexpr (TPR == 32) {
    // the warps of the block add their sums one after the other, over the ring, which nobody reads any more
    float* sums = reinterpret_cast<float*>(scratch);
    __syncthreads();
    for (int turn = 0; turn < rows; ++turn) {
      if (sub == turn) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int c = (i * TPR + t) * VEC;
          if (c < a.D) {
#pragma unroll
            for (int e = 0; e < P2; ++e) {
              float2* pw = reinterpret_cast<float2*>(sums + c + 2 * e);
              float2* pb = reinterpret_cast<float2*>(sums + a.D + c + 2 * e);
              const float2 w = turn ? *pw : make_float2(0.f, 0.f), b = turn ? *pb : make_float2(0.f, 0.f);
              *pw = make_float2(w.x + dw[i][e].v.x, w.y + dw[i][e].v.y);
              *pb = make_float2(b.x + db[i][e].v.x, b.y + db[i][e].v.y);
            }
          }
        }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < 2 * a.D; c += T0) out[c] = sums[c];
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * VEC;
      if (c < a.D) {
#pragma unroll
        for (int e = 0; e < P2; ++e) {
          *reinterpret_cast<float2*>(out + c + 2 * e) = dw[i][e].v;
          *reinterpret_cast<float2*>(out + a.D + c + 2 * e) = db[i][e].v;
        }
      }
    }
  }
}

// The same without 16-byte access (odd widths and strides, unaligned addresses): one value per piece, rows as they come.
template <class T, class W, int NV, int TPR>
__global__ void __launch_bounds__(TPR == 32 ? 384 : TPR) norm_bwd_odd_kernel(const NormDev a) {
  extern __shared__ float odd_sums[];  // TPR == 32 with partial sums: 2 * D floats
  __shared__ float2 sm[2 * (TPR / 32)];
  griddep_wait();
  griddep_launch();
  const int t = TPR == 32 ? threadIdx.x & 31 : threadIdx.x;
  const int sub = TPR == 32 ? threadIdx.x >> 5 : 0;
  const int rows = TPR == 32 ? blockDim.x >> 5 : 1;
  const float inv_d = 1.f / static_cast<float>(a.D);
  float w[NV], dw[NV], db[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = i * TPR + t;
    Piece<W, 1> p;
    if (a.has_w && c < a.D) p.ld(static_cast<const W*>(a.w) + c);
    w[i] = a.has_w && c < a.D ? p.get(0) : 1.f;
    dw[i] = db[i] = 0.f;
  }
  int slot = 0;
  for (long long row = static_cast<long long>(blockIdx.x) * rows + sub; row < a.M; row += static_cast<long long>(gridDim.x) * rows) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* g = static_cast<const T*>(a.dy) + row * a.ld_dy;
    Piece<T, 1> px[NV], pg[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = i * TPR + t;
      if (c < a.D) px[i].ld(x + c), pg[i].ld(g + c);
      else px[i].zero(), pg[i].zero();
    }
    const float2 st = __ldg(a.stats + row);
    const float r = st.y, off = -st.x * st.y;
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const float gv = pg[i].get(0), xh = fmaf(px[i].get(0), r, off), h = gv * w[i];  // gv is 0 behind the row's end
      s1 += h;
      s2 = fmaf(h, xh, s2);
      dw[i] = fmaf(gv, xh, dw[i]);
      db[i] += gv;
    }
    if (!a.dx) continue;  // the same for every thread
    const float2 s = row_sum2<TPR>(s1, s2, sm, slot);
    slot ^= 1;
    const float c1 = s.x * inv_d, c2 = s.y * inv_d;
    T* dx = static_cast<T*>(a.dx) + row * a.ld_dx;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = i * TPR + t;
      if (c < a.D) {
        const float o[1] = {r * (pg[i].get(0) * w[i] - c1 - fmaf(px[i].get(0), r, off) * c2)};
        px[i].set(o);
        px[i].st(dx + c);
      }
    }
  }
  if (!a.partial) return;
  float* out = a.partial + static_cast<long long>(blockIdx.x) * 2 * a.D;
  if constexpr (TPR == 32) {
    for (int turn = 0; turn < rows; ++turn) {
      if (sub == turn) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int c = i * TPR + t;
          if (c < a.D) {
            odd_sums[c] = (turn ? odd_sums[c] : 0.f) + dw[i];
            odd_sums[a.D + c] = (turn ? odd_sums[a.D + c] : 0.f) + db[i];
          }
        }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < 2 * a.D; c += blockDim.x) out[c] = odd_sums[c];
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = i * TPR + t;
      if (c < a.D) out[c] = dw[i], out[a.D + c] = db[i];
    }
  }
}

// Wide rows, backward: dx in passes over the row; the gradients of w and b by norm_wide_grads_kernel.
template <class T, class W>
__global__ void __launch_bounds__(512) norm_bwd_wide_kernel(const NormDev a) {
  __shared__ float2 sm[32];
  griddep_wait();
  griddep_launch();
  const float inv_d = 1.f / static_cast<float>(a.D);
  int slot = 0;
  for (long long row = blockIdx.x; row < a.M; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* g = static_cast<const T*>(a.dy) + row * a.ld_dy;
    T* dx = static_cast<T*>(a.dx) + row * a.ld_dx;
    const float2 st = __ldg(a.stats + row);
    Piece<T, 1> px, pg;
    Piece<W, 1> pw;
    float s1 = 0.f, s2 = 0.f;
    for (int c = threadIdx.x; c < a.D; c += 512) {
      px.ld(x + c), pg.ld(g + c);
      if (a.has_w) pw.ld(static_cast<const W*>(a.w) + c);
      const float h = a.has_w ? pg.get(0) * pw.get(0) : pg.get(0);
      s1 += h;
      s2 = fmaf(h, (px.get(0) - st.x) * st.y, s2);
    }
    const float2 s = row_sum2<512>(s1, s2, sm, slot);
    slot ^= 1;
    for (int c = threadIdx.x; c < a.D; c += 512) {
      px.ld(x + c), pg.ld(g + c);
      if (a.has_w) pw.ld(static_cast<const W*>(a.w) + c);
      const float h = a.has_w ? pg.get(0) * pw.get(0) : pg.get(0);
      const float o[1] = {st.y * (h - s.x * inv_d - (px.get(0) - st.x) * st.y * (s.y * inv_d))};
      px.set(o);
      px.st(dx + c);
    }
  }
}

// partial[blockIdx.y] = sums over every gridDim.y-th row of one column per thread.
template <class T>
__global__ void __launch_bounds__(256) norm_wide_grads_kernel(const NormDev a) {
  griddep_wait();
  griddep_launch();
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.D) return;
  float dw = 0.f, db = 0.f;
  Piece<T, 1> px, pg;
  for (long long row = blockIdx.y; row < a.M; row += gridDim.y) {
    px.ld(static_cast<const T*>(a.x) + row * a.ldx + c);
    pg.ld(static_cast<const T*>(a.dy) + row * a.ld_dy + c);
    const float2 st = __ldg(a.stats + row);
    dw = fmaf(pg.get(0), (px.get(0) - st.x) * st.y, dw);
    db += pg.get(0);
  }
  float* out = a.partial + static_cast<long long>(blockIdx.y) * 2 * a.D;
  out[c] = dw, out[a.D + c] = db;
}

// ---------------------------------------------------------------- plans
struct NormPlan {
  int vec, nv, tpr;  // tpr 0: the kernels for wide rows
};

// Threads per row: a warp where the row fits in its registers (five pieces per lane), so that no barrier joins a row's
// sums; else 128 or 512 threads with up to four pieces.
NormPlan norm_plan(int D, int dtype, bool wide_access) {
  const int vec = wide_access ? (dtype == POM_BF16 ? 8 : 4) : 1;
  const int64_t pieces = ceil_div(D, vec);
  if (pieces <= 32 * 5) return NormPlan{vec, static_cast<int>(ceil_div(pieces, 32)), 32};
  if (pieces <= 128 * 4) return NormPlan{vec, static_cast<int>(ceil_div(pieces, 128)), 128};
  if (pieces <= 512 * 4) return NormPlan{vec, static_cast<int>(ceil_div(pieces, 512)), 512};
  return NormPlan{1, 0, 0};
}

constexpr int kMaxBwdSmem = 200 * 1024;
constexpr int kFwdWarps = 8, kBwdWarps = 12, kWideSplits = 64;

int bwd_blocks(int64_t M, const NormPlan& p) {
  const int64_t want = p.tpr == 32 ? ceil_div(M, kBwdWarps) : M;
  const int64_t cap = static_cast<int64_t>(sm_count()) * (p.tpr == 128 ? 3 : 1);
  return static_cast<int>(want < cap ? want : cap);
}

template <class T, class W, int VEC, int NV, int TPR>
int launch_norm(const NormDev& d, bool bwd, int blocks, cudaStream_t st) {
  cudaError_t e;
  if (bwd) {
    const int threads = TPR == 32 ? 32 * kBwdWarps : TPR;
    const size_t sums = TPR == 32 && d.partial ? 2 * static_cast<size_t>(d.D) * sizeof(float) : 0;
    if constexpr (VEC > 1) {
      const int ring = NV * TPR * VEC * 4 + kBwdStages<TPR> * 2 * NV * threads * 16;
      const int smem = static_cast<int>(sums) > ring ? static_cast<int>(sums) : ring;
      static_assert(NV * TPR * VEC * 4 + kBwdStages<TPR> * 2 * NV * (TPR == 32 ? 32 * kBwdWarps : TPR) * 16 <= kMaxBwdSmem);
      static std::atomic<uint64_t> attr_set{0};
      auto kern = norm_bwd_kernel<T, W, NV, TPR>;
      const int rc = once_per_device(attr_set, [&] {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxBwdSmem) != cudaSuccess) {
          (void)cudaGetLastError();
          return static_cast<int>(POM_ERR_CUDA);
        }
        return static_cast<int>(POM_OK);
      });
      if (rc) return rc;
      e = launch_pdl(kern, dim3(blocks), dim3(threads), smem, st, d);
    } else {
      e = launch_pdl(norm_bwd_odd_kernel<T, W, NV, TPR>, dim3(blocks), dim3(threads), sums, st, d);
    }
  } else {
    const int threads = TPR == 32 ? 32 * kFwdWarps : TPR;
    const int64_t want = ceil_div(d.M, TPR == 32 ? kFwdWarps : 1), cap = 32ll * sm_count();
    e = launch_pdl(norm_fwd_kernel<T, W, VEC, NV, TPR>, dim3(static_cast<unsigned>(want < cap ? want : cap)), dim3(threads),
                   0, st, d);
  }
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return POM_ERR_CUDA;
  }
  count_launch();
  return POM_OK;
}

template <class T, class W, int VEC>
int norm_any(const NormDev& d, const NormPlan& p, bool bwd, int blocks, cudaStream_t st) {
#define POM_NORM(NV_, TPR_) \
  if (p.nv == NV_ && p.tpr == TPR_) return launch_norm<T, W, VEC, NV_, TPR_>(d, bwd, blocks, st);
  POM_NORM(1, 32) POM_NORM(2, 32) POM_NORM(3, 32) POM_NORM(4, 32) POM_NORM(5, 32)
  POM_NORM(2, 128) POM_NORM(3, 128) POM_NORM(4, 128)
  POM_NORM(2, 512) POM_NORM(3, 512) POM_NORM(4, 512)
#undef POM_NORM
  return POM_ERR_UNSUPPORTED;
}

template <class T, class W>
int norm_wide(const NormDev& d, bool bwd, cudaStream_t st) {
  const int64_t cap = 4ll * sm_count();
  const dim3 grid(static_cast<unsigned>(d.M < cap ? d.M : cap));
  cudaError_t e = cudaSuccess;
  if (!bwd) {
    e = launch_pdl(norm_fwd_wide_kernel<T, W>, grid, dim3(512), 0, st, d);
    count_launch();
  } else {
    if (d.dx) e = launch_pdl(norm_bwd_wide_kernel<T, W>, grid, dim3(512), 0, st, d), count_launch();
    if (e == cudaSuccess && d.partial) {
      const dim3 g2(static_cast<unsigned>(ceil_div(d.D, 256)), static_cast<unsigned>(d.M < kWideSplits ? d.M : kWideSplits));
      e = launch_pdl(norm_wide_grads_kernel<T>, g2, dim3(256), 0, st, d);
      count_launch();
    }
  }
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return POM_ERR_CUDA;
  }
  return POM_OK;
}

int run_norm(const NormDev& d, const NormPlan& p, int dtype, int wdtype, bool bwd, int blocks, cudaStream_t st) {
  if (!d.has_w) wdtype = dtype;
  using B = __nv_bfloat16;
  if (dtype == POM_BF16 && wdtype == POM_BF16)
    return !p.tpr ? norm_wide<B, B>(d, bwd, st) : p.vec == 8 ? norm_any<B, B, 8>(d, p, bwd, blocks, st) : norm_any<B, B, 1>(d, p, bwd, blocks, st);
  if (dtype == POM_BF16)
    return !p.tpr ? norm_wide<B, float>(d, bwd, st) : p.vec == 8 ? norm_any<B, float, 8>(d, p, bwd, blocks, st) : norm_any<B, float, 1>(d, p, bwd, blocks, st);
  return !p.tpr ? norm_wide<float, float>(d, bwd, st) : p.vec == 4 ? norm_any<float, float, 4>(d, p, bwd, blocks, st) : norm_any<float, float, 1>(d, p, bwd, blocks, st);
}

int check_norm(const pom_layer_norm_args* a) {
  if (!a || !a->x) return POM_ERR_NULL;
  if (a->M <= 0 || a->D <= 0) return POM_ERR_BAD_SHAPE;
  if (a->D > (1 << 24)) return POM_ERR_TOO_LARGE;
  if (a->dtype != POM_BF16 && a->dtype != POM_F32) return POM_ERR_UNSUPPORTED;
  if (a->wdtype != POM_F32 && (a->wdtype != POM_BF16 || a->dtype != POM_BF16)) return POM_ERR_UNSUPPORTED;
  if (a->bias && !a->weight) return POM_ERR_UNSUPPORTED;
  if (a->ldx < a->D) return POM_ERR_BAD_STRIDE;
  if (reinterpret_cast<uintptr_t>(a->stats) & 7u) return POM_ERR_BAD_ALIGN;
  return POM_OK;
}

// 16-byte access to every row of these operands.
bool wide_rows(const pom_layer_norm_args* a, std::initializer_list<const void*> ptrs, std::initializer_list<int64_t> lds) {
  const int per = a->dtype == POM_BF16 ? 8 : 4;
  if (a->D % per) return false;
  for (const void* p : ptrs)
    if (p && !aligned16(p)) return false;
  for (int64_t l : lds)
    if (l % per) return false;
  return true;
}

NormPlan bwd_plan(const pom_layer_norm_args* a) {
  return norm_plan(a->D, a->dtype, wide_rows(a, {a->x, a->dy, a->dx, a->weight}, {a->ldx, a->ld_dy, a->dx ? a->ld_dx : 0}));
}

int partial_rows(const pom_layer_norm_args* a, const NormPlan& p) {
  return p.tpr ? bwd_blocks(a->M, p) : static_cast<int>(a->M < kWideSplits ? a->M : kWideSplits);
}

NormDev norm_dev(const pom_layer_norm_args* a) {
  NormDev d;
  d.x = a->x, d.y = a->y;
  d.has_w = a->weight != nullptr, d.has_b = a->bias != nullptr;
  d.w = a->weight ? a->weight : a->x, d.b = a->bias ? a->bias : d.w;
  d.stats = reinterpret_cast<float2*>(a->stats);
  d.dy = a->dy, d.dx = a->dx, d.partial = nullptr;
  d.M = a->M, d.ldx = a->ldx, d.ldy = a->ldy, d.ld_dy = a->ld_dy, d.ld_dx = a->ld_dx;
  d.D = a->D, d.eps = a->eps;
  return d;
}

}  // namespace

extern "C" {

int pom_layer_norm_fwd(const pom_layer_norm_args* a, void* stream) {
  int rc = check_norm(a);
  if (rc) return rc;
  if (!a->y) return POM_ERR_NULL;
  if (a->ldy < a->D) return POM_ERR_BAD_STRIDE;
  const NormPlan p = norm_plan(a->D, a->dtype, wide_rows(a, {a->x, a->y, a->weight, a->bias}, {a->ldx, a->ldy}));
  return run_norm(norm_dev(a), p, a->dtype, a->wdtype, false, 0, static_cast<cudaStream_t>(stream));
}

uint64_t pom_layer_norm_bwd_workspace(const pom_layer_norm_args* a) {
  if (check_norm(a) || (!a->dweight && !a->dbias)) return 0;
  return static_cast<uint64_t>(partial_rows(a, bwd_plan(a))) * 2 * static_cast<uint64_t>(a->D) * sizeof(float);
}

int pom_layer_norm_bwd(const pom_layer_norm_args* a, void* stream) {
  int rc = check_norm(a);
  if (rc) return rc;
  const bool grads = a->dweight || a->dbias;
  if (!a->dy || !a->stats || (grads && !a->workspace)) return POM_ERR_NULL;
  if (!a->dx && !grads) return POM_OK;
  if (a->ld_dy < a->D || (a->dx && a->ld_dx < a->D)) return POM_ERR_BAD_STRIDE;
  if (!aligned16(a->workspace)) return POM_ERR_BAD_ALIGN;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const NormPlan p = bwd_plan(a);
  NormDev d = norm_dev(a);
  d.partial = grads ? static_cast<float*>(a->workspace) : nullptr;
  const int blocks = bwd_blocks(a->M, p);
  if ((rc = run_norm(d, p, a->dtype, a->wdtype, true, blocks, st))) return rc;
  if (grads &&
      (rc = sum_rows(d.partial, partial_rows(a, p), 2 * a->D, a->D, a->wdtype, a->dweight, a->dbias, st)))
    return rc;
  return check_launch();
}
}  // extern "C"
