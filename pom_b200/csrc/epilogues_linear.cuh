// Epilogue of the linear operator on the tcgen05 GEMM engine: y = act(acc + bias) + residual, and, for a backward pass,
// the slope act'(acc + bias) beside it.
//
// The slope is kept instead of the pre-activation: both cost one bf16 per element, but with the slope the backward pass
// is a product (dz = dy * slope) where the pre-activation would need the derivative again from its rounded value.
// Rounding the slope to bf16 (half a step, 2^-9 of its value) puts the same relative error into dz as rounding dz itself,
// which the tensor cores need anyway.
#pragma once
#include "epilogues.cuh"
#include "f32x2.cuh"
#include "linear_math.cuh"

namespace pomk {

// 32 values of a row: v becomes act(v), and with SLOPE ps the packed act'(v).
template <int ACT, bool SLOPE>
__device__ __forceinline__ void linear_act32(float (&v)[32], uint32_t (&ps)[16]) {
#pragma unroll
  for (int i = 0; i < 32; i += 2) {
    float s0, s1;
    v[i] = linear_act<SLOPE, true>(ACT, v[i], s0);
    v[i + 1] = linear_act<SLOPE, true>(ACT, v[i + 1], s1);
    if (SLOPE) ps[i / 2] = pack_bf16x2(s0, s1);
  }
}

// gelu of 32 values in packed pairs: the arithmetic of linear_act<SLOPE, true>.
template <bool SLOPE>
__device__ __forceinline__ void gelu32(float (&v)[32], uint32_t (&ps)[16]) {
#pragma unroll
  for (int i = 0; i < 32; i += 2) {
    const F2 z(v[i], v[i + 1]);
    const F2 d = fma2(F2(fabsf(z.v.x), fabsf(z.v.y)), F2(0.2316418882f), F2(1.f));
    const F2 t(fast_rcp(d.v.x), fast_rcp(d.v.y));
    const F2 w = mul2(mul2(z, F2(-0.72134752044f)), z);
    const F2 e(fast_exp2(w.v.x), fast_exp2(w.v.y));
    F2 q = fma2(F2(0.5307027145f), t, F2(-0.7265760135f));
    q = fma2(q, t, F2(0.7107068705f));
    q = fma2(q, t, F2(-0.142248368f));
    q = fma2(q, t, F2(0.127414796f));
    q = mul2(q, mul2(t, e));
    const F2 up = fma2(q, F2(-1.f), F2(1.f));
    const F2 phi(z.v.x < 0.f ? q.v.x : up.v.x, z.v.y < 0.f ? q.v.y : up.v.y);
    if (SLOPE) {
      const F2 s = fma2(mul2(z, F2(0.3989422804014327f)), e, phi);
      ps[i / 2] = pack_bf16x2(s.v.x, s.v.y);
    }
    const F2 y = mul2(z, phi);
    v[i] = y.v.x, v[i + 1] = y.v.y;
  }
}

template <bool SLOPE>
__device__ __forceinline__ void linear_act32(int act, float (&v)[32], uint32_t (&ps)[16]) {
  switch (act) {
    case POM_ACT_GELU: gelu32<SLOPE>(v, ps); break;
    case POM_ACT_GELU_TANH: linear_act32<POM_ACT_GELU_TANH, SLOPE>(v, ps); break;
    case POM_ACT_SILU: linear_act32<POM_ACT_SILU, SLOPE>(v, ps); break;
    case POM_ACT_RELU: linear_act32<POM_ACT_RELU, SLOPE>(v, ps); break;
    default: linear_act32<POM_ACT_NONE, SLOPE>(v, ps); break;
  }
}

template <bool RES>
struct EpiLinear {
  struct Params {
    const void* bias;  // (N) bf16 or fp32, or null
    int bias_f32;
    int act;
    int save_slope;  // maps.out0 = slope; maps.out1 = y; maps.in0 = residual
  };
  static constexpr int kSmemBytes = 2 * 256 * 4;  // double-buffered bias
  // per warp: [slope or y][y], with a residual [residual in][y][slope]
  static constexpr int kStageBytes = RES ? 6144 : 4096;
  static constexpr bool kStager = false;
  template <int BN>
  static constexpr int smem_bytes() { return kSmemBytes; }

  static __device__ __forceinline__ void fetch(const EpiMaps& maps, const TileCtx& t, EpiIO& io, int quarter, int lane,
                                               int col) {
    if (lane == 0) {
      mbar_expect_tx(io.bar, 32 * 64);
      tma_load_3d(io.buf0, &maps.in0, io.bar, col, t.row0 + quarter * 32, t.b);
    }
  }

  template <int BN>
  static __device__ __forceinline__ void prologue(const Params& p, const EpiMaps& maps, const GemmGeom& g,
                                                  const TileCtx& t, int warp_in_epi, int epi_tid, float* scratch,
                                                  EpiIO& io, int iter) {
    if constexpr (RES) {
      const int half = warp_in_epi >> 2, quarter = (warp_in_epi + 2) & 3;
      const int col = t.col0 + half * 32;
      if (col < g.n_cols) fetch(maps, t, io, quarter, epi_tid & 31, col);
    }
    float* cst = scratch + (iter & 1) * 256;
    for (int j = epi_tid; j < BN; j += kEpiThreads) {
      const int col = t.col0 + j;
      float v = 0.f;
      if (p.bias && col < g.n_cols)
        v = p.bias_f32 ? __ldg(static_cast<const float*>(p.bias) + col)
                       : __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(p.bias) + col));
      cst[j] = v;
    }
    named_bar_sync(kEpiBarrier, kEpiThreads);
  }

  template <int BN>
  static __device__ __forceinline__ void run(const Params& p, const EpiMaps& maps, const GemmGeom& g, const TileCtx& t,
                                             uint32_t tmem_acc, int quarter, int lane, int half, int, float* scratch,
                                             EpiIO& io, int iter) {
    const float* cst = scratch + (iter & 1) * 256;
    const int y = t.row0 + quarter * 32;
    uint8_t* const base = io.buf0;
    // the alternation starts anew with every tile, and a tile may have an odd number of chunks
    if (lane == 0) bulk_wait_read<0>();
    int flip = 0;
    bool alive = true;
#pragma unroll 1
    for (int c = half; c < BN / 32; c += kEpiColSplit) {
      const int col = t.col0 + c * 32;
      if (col >= g.n_cols) break;  // warp-uniform; the load of this chunk was not started either
      float v[32];
      uint32_t pk[16];
      tmem_ld32(tmem_acc + c * 32, v);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 32; i += 4) {
        const float4 b = *reinterpret_cast<const float4*>(cst + c * 32 + i);
        v[i] += b.x, v[i + 1] += b.y, v[i + 2] += b.z, v[i + 3] += b.w;
      }
      if (p.save_slope) {
        linear_act32<true>(p.act, v, pk);
        if (t.rows_valid > 0) store_block<1>(RES ? base + 4096 : base, &maps.out0, pk, lane, col, y, t.b);
      } else {
        linear_act32<false>(p.act, v, pk);
      }
      if constexpr (RES) {
        float r[32];
        if (alive) alive = mbar_wait(io.bar, io.load_phase, io.abort_flag, io.status, kStatusEpilogueTimeout);
        alive = __all_sync(0xffffffffu, alive);
        io.load_phase ^= 1u;
        read_block(base, lane, r);
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] += r[i];
        __syncwarp();  // every lane has its residual row: the block may be refilled
        const int ncol = t.col0 + (c + kEpiColSplit) * 32;
        if (alive && c + kEpiColSplit < BN / 32 && ncol < g.n_cols) fetch(maps, t, io, quarter, lane, ncol);
      }
      pack32(v, pk);
      if (t.rows_valid > 0) {
        // with a slope the two stores use one block each; without one, y alternates between two blocks
        uint8_t* out = RES ? base + (p.save_slope || !flip ? 2048 : 4096) : (p.save_slope || flip ? base + 2048 : base);
        store_block<1>(out, &maps.out1, pk, lane, col, y, t.b);
      }
      flip ^= 1;
    }
  }
};

}  // namespace pomk
