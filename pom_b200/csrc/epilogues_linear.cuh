// Epilogue of the linear operator on the tcgen05 GEMM engine: y = act(z) + residual with z = acc + bias, and, for a backward
// pass, z beside it.
//
// z is kept rounded to bf16 and its slope formed again in the backward pass: an error of 2^-9 in z moves the slope by that
// times |z| act''(z), a quarter of what rounding the slope itself would do.  What remains is the rounding of dz, which the
// tensor cores need.
//
// 32768 x 1152 -> 4608 with gelu and z: 295 us (268 without an activation, the product's own time; with erff and expf per
// element 397), so the activation's arithmetic, not the stores, is what the product waits for.
#pragma once
#include "epilogues.cuh"
#include "linear_math.cuh"

namespace pomk {

template <int ACT, int LEN>
__device__ __forceinline__ void linear_act_row(float (&v)[LEN]) {
#pragma unroll
  for (int i = 0; i < LEN; i += 2) {
    const F2 y = linear_act2<true>(ACT, F2(v[i], v[i + 1]));
    v[i] = y.v.x, v[i + 1] = y.v.y;
  }
}

// Adjacent values of a row; the choice of the activation stands outside their loop.
template <int LEN>
__device__ __forceinline__ void linear_act_row(int act, float (&v)[LEN]) {
  switch (act) {
    case POM_ACT_GELU: linear_act_row<POM_ACT_GELU>(v); break;
    case POM_ACT_GELU_TANH: linear_act_row<POM_ACT_GELU_TANH>(v); break;
    case POM_ACT_SILU: linear_act_row<POM_ACT_SILU>(v); break;
    case POM_ACT_RELU: linear_act_row<POM_ACT_RELU>(v); break;
    default: break;
  }
}

template <bool RES>
struct EpiLinear {
  struct Params {
    const void* bias;  // (N) bf16 or fp32; has_bias 0: an address that may be read
    int has_bias, bias_f32;
    int act;
    int save_z;  // maps.out0 = z; maps.out1 = y; maps.in0 = residual
  };
  static constexpr int kSmemBytes = 2 * 256 * 4;  // double-buffered bias
  // per warp: [z or y][y], with a residual [residual in][y][z or y]
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
      if (p.has_bias && col < g.n_cols)
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
      if (p.save_z) {
        pack32(v, pk);
        if (t.rows_valid > 0) store_block<1>(RES ? base + 4096 : base, &maps.out0, pk, lane, col, y, t.b);
      }
      linear_act_row(p.act, v);
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
        // with z the two stores use one block each; without it, y alternates between two blocks
        uint8_t* out = RES ? base + (p.save_z || !flip ? 2048 : 4096) : (p.save_z || flip ? base + 2048 : base);
        store_block<1>(out, &maps.out1, pk, lane, col, y, t.b);
      }
      flip ^= 1;
    }
  }
};

}  // namespace pomk
