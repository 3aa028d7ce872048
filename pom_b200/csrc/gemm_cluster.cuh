// bf16 product with few output tiles and a long K: a cluster of CTAs shares one 128 x BN tile, each CTA takes a run of the
// k-blocks, and the partial tiles are added through distributed shared memory.
//
// One CTA's main loop waits for its operands: a 64-long k-block of a 128 x 128 tile is 32 KB, and an SM takes in about 64
// bytes a cycle (0.285 us a block, whatever else runs), so a product of few tiles and a long K leaves most SMs idle
// while a few of them read.  A cluster of `size` CTAs divides that time by `size`.  Every CTA owns BN / size columns of the
// result: it sends the other columns of its partial tile to their owners (st.shared::cluster, 512 adjacent bytes a warp: with
// the rows apart, the same stores took 4 us instead of 1), and after one cluster barrier adds what it has received to its own
// accumulator, in the order of the ranks: the same bits on every run.  Then bias, activation and residual, which
// were fetched while the main loop ran, and bulk stores of 32 x 32 blocks (16 columns: from registers).
//
// Roles and waits as in gemm_sm100.cuh: warp 0 loads, warp 1 issues the MMAs, warps 2 to 9 are the epilogue; every wait on
// a barrier in shared memory is bounded, and every thread reaches both cluster barriers whatever happened before.
#pragma once
#include "epilogues_linear.cuh"
#include "gemm_launch.cuh"

namespace pomk {

struct ClusterDev {
  const void* bias;  // (N) bf16 or fp32
  const __nv_bfloat16* residual;
  int has_bias, has_residual;  // 0: set to the first operand by cluster_product, an address that may be read
  __nv_bfloat16* y;
  __nv_bfloat16* z;  // contiguous, or null
  long long ldr, ldy;
  int bias_f32, act;
  int M, N, m_tiles, k_blocks;
};

constexpr int kClusterThreads = 32 * (2 + kEpiWarps);
constexpr int kClusterMax = 8;

template <int BN>
struct ClusterSmem {
  static constexpr int kStageBytes = (kBM + BN) * kBK * 2;
  static constexpr int kStages = BN == 128 ? 5 : 3;
  // partial tiles of the other ranks: (size - 1) / size of 128 x BN fp32 (BN 256: at most two CTAs)
  static constexpr int kRecvBytes = BN == 128 ? 56 * 1024 : 64 * 1024;
  static constexpr int kBiasBytes = 128 * 4;  // of the columns that this CTA finishes
  static constexpr int kBytes = kStages * kStageBytes + kRecvBytes + kBiasBytes + 256 + 1024;
};

__device__ __forceinline__ void st_cluster(uint32_t addr, float a, float b, float c, float d) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}

// Columns 4 j .. 4 j + 3 of row `row` of a partial tile: the rows of a warp lie side by side.
__device__ __forceinline__ uint32_t recv_offset(int row, int j) { return static_cast<uint32_t>((j * kBM + row) * 16); }

template <int BN, bool B_MN>  // A: K-major
__global__ void __launch_bounds__(kClusterThreads, 1)
gemm_cluster_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ CUtensorMap tmY, const __grid_constant__ CUtensorMap tmZ, const ClusterDev a,
                    int* __restrict__ status) {
  using S = ClusterSmem<BN>;
  constexpr int kABytes = kBM * kBK * 2;
  constexpr uint32_t kIdesc = make_idesc_bf16(BN, false, B_MN);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* recv = tiles + S::kStages * S::kStageBytes;
  float* bias_sm = reinterpret_cast<float*>(recv + S::kRecvBytes);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(recv + S::kRecvBytes + S::kBiasBytes);
  uint64_t* empty_bar = full_bar + S::kStages;
  uint64_t* done_bar = empty_bar + S::kStages;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(done_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t size;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
  const uint32_t rank = cluster_ctarank();
  const int tile = blockIdx.x / size;
  const int row0 = (tile % a.m_tiles) * kBM, col0 = (tile / a.m_tiles) * BN;
  const int kb0 = rank * a.k_blocks / size, kb1 = (rank + 1) * a.k_blocks / size;  // at least one each
  const int slice = BN / size;  // columns this CTA finishes: 16, 32, 64 or 128

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(done_bar, 1);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 1) {
    tmem_alloc(tmem_holder, BN);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // every CTA of the cluster runs: its shared memory may be written
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  griddep_wait();
  griddep_launch();

  bool ok = true;
  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&empty_bar[stage], phase ^ 1u, abort_flag, status, kStatusProducerTimeout)) {
          ok = false;
          break;
        }
        uint8_t* sa = tiles + stage * S::kStageBytes;
        uint8_t* sb = sa + kABytes;
        mbar_expect_tx(&full_bar[stage], S::kStageBytes);
        tma_load_3d(sa, &tmA, &full_bar[stage], kb * kBK, row0, 0);
        if constexpr (!B_MN) {
          tma_load_3d(sb, &tmB, &full_bar[stage], kb * kBK, col0, 0);
        } else {
#pragma unroll
          for (int j = 0; j < BN / 64; ++j)
            tma_load_3d(sb + j * (kBK * 128), &tmB, &full_bar[stage], col0 + j * 64, kb * kBK, 0);
        }
        if (++stage == S::kStages) stage = 0, phase ^= 1u;
      }
      if (!ok)
        for (int i = 0; i < 64; ++i) __nanosleep(2000);  // loads in flight land before the CTA retires
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&full_bar[stage], phase, abort_flag, status, kStatusMmaTimeout)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t sa = smem_u32(tiles + stage * S::kStageBytes), sb = sa + kABytes;
#pragma unroll
        for (int k16 = 0; k16 < kBK / 16; ++k16) {
          const uint64_t da = make_smem_desc(sa + k16 * 32, 16, 1024);
          const uint64_t db = B_MN ? make_smem_desc(sb + k16 * 2048, kBK * 128, 1024) : make_smem_desc(sb + k16 * 32, 16, 1024);
          umma_bf16(tmem, da, db, kIdesc, (kb > kb0 || k16 > 0) ? 1u : 0u);
        }
        umma_commit(&empty_bar[stage]);
        if (++stage == S::kStages) stage = 0, phase ^= 1u;
      }
      if (ok) umma_commit(done_bar);
      else
        for (int i = 0; i < 64; ++i) __nanosleep(2000);
    }
  }
  const int quarter = warp & 3, half = (warp - 2) >> 2;  // epilogue warps: TMEM lanes of this warp, and which pieces
  const int row = quarter * 32 + lane;
  const uint32_t acc = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
  const long long r = row0 + row;
  const int first = col0 + static_cast<int>(rank) * slice;  // first column that this CTA finishes
  const int width = slice < 32 ? slice : 32;                 // columns of a chunk; a warp takes chunks half, half + 2, ...
  // residual of the eight columns at `at` of this CTA's slice (N is a multiple of 8)
  auto residual = [&](int at) {
    if (a.has_residual && r < a.M && at < slice && first + at < a.N)
      return __ldg(reinterpret_cast<const uint4*>(a.residual + r * a.ldr + first + at));
    return make_uint4(0, 0, 0, 0);
  };
  uint4 res = make_uint4(0, 0, 0, 0);
  if (warp >= 2) {
    const int e = threadIdx.x - 64;
    if (e < slice) {
      float b = 0.f;
      if (a.has_bias && first + e < a.N)
        b = a.bias_f32 ? __ldg(static_cast<const float*>(a.bias) + first + e)
                       : __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(a.bias) + first + e));
      bias_sm[e] = b;
    }
    res = residual(half * width);
    ok = mbar_wait(done_bar, 0, abort_flag, status, kStatusEpilogueTimeout);
    ok = __all_sync(0xffffffffu, ok);
    tc_fence_after();
    if (ok) {
      // 32 columns at a time, each 16 of them to the rank that owns them
      const uint32_t recv0 = smem_u32(recv);
#pragma unroll 1
      for (int c = half; c < BN / 32; c += 2) {
        float v[32];
        tmem_ld32(acc + c * 32, v);
        tmem_ld_wait();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int col = c * 32 + h * 16;
          const uint32_t owner = col / slice;
          if (owner != rank) {
            const uint32_t slot = rank < owner ? rank : rank - 1;
            const uint32_t dst = map_to_cta(recv0, owner) + slot * (kBM * slice * 4);
            const int j0 = (col - static_cast<int>(owner) * slice) / 4;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int k = h * 16 + 4 * j;
              st_cluster(dst + recv_offset(row, j0 + j), v[k], v[k + 1], v[k + 2], v[k + 3]);
            }
          }
        }
      }
    }
  }
  __syncwarp();
  cluster_sync_all();  // every partial tile has arrived; nobody writes to another CTA after this
  if (warp >= 2 && ok) {
    uint8_t* buf = tiles + (warp - 2) * 8192;  // the operand tiles have been read: two blocks for each of this warp's chunks
    const int top = row0 + quarter * 32;
#pragma unroll 1
    for (int at0 = half * width; at0 < slice && first + at0 < a.N; at0 += 2 * width, buf += 4096) {  // warp-uniform
#pragma unroll 1
      for (int j = 0; j < width / 8; ++j) {
        const int at = at0 + 8 * j;
        float own[8], v[8];
        tmem_ld8(acc + rank * slice + at, own);
        const uint4 mine = res;
        res = residual(j + 1 < width / 8 ? at + 8 : at0 + 2 * width);  // of the columns after these
        tmem_ld_wait();
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = 0.f;
        for (uint32_t s = 0; s < size; ++s) {
          const uint8_t* src = recv + (s < rank ? s : s - 1) * (kBM * slice * 4);
          float4 p = make_float4(own[0], own[1], own[2], own[3]), q = make_float4(own[4], own[5], own[6], own[7]);
          if (s != rank) {
            p = *reinterpret_cast<const float4*>(src + recv_offset(row, at / 4));
            q = *reinterpret_cast<const float4*>(src + recv_offset(row, at / 4 + 1));
          }
          v[0] += p.x, v[1] += p.y, v[2] += p.z, v[3] += p.w;
          v[4] += q.x, v[5] += q.y, v[6] += q.z, v[7] += q.w;
        }
#pragma unroll
        for (int k = 0; k < 8; k += 4) {
          const float4 b = *reinterpret_cast<const float4*>(bias_sm + at + k);
          v[k] += b.x, v[k + 1] += b.y, v[k + 2] += b.z, v[k + 3] += b.w;
        }
        const uint4 pz = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
        linear_act_row(a.act, v);
        const uint32_t w[4] = {mine.x, mine.y, mine.z, mine.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[2 * e] += __uint_as_float(w[e] << 16);
          v[2 * e + 1] += __uint_as_float(w[e] & 0xffff0000u);
        }
        const uint4 py = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
        if (width == 32) {
          *reinterpret_cast<uint4*>(buf + swz64(lane, j)) = py;
          if (a.z) *reinterpret_cast<uint4*>(buf + 2048 + swz64(lane, j)) = pz;
        } else if (r < a.M && first + at < a.N) {
          *reinterpret_cast<uint4*>(a.y + r * a.ldy + first + at) = py;
          if (a.z) *reinterpret_cast<uint4*>(a.z + r * a.N + first + at) = pz;
        }
        __syncwarp();  // the next tensor-memory load wants the whole warp
      }
      if (width == 32 && top < a.M) {  // blocks are clipped at the last row and column
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store_3d(&tmY, buf, first + at0, top, 0);
          if (a.z) tma_store_3d(&tmZ, buf + 2048, first + at0, top, 0);
          bulk_commit();
        }
      }
    }
    if (lane == 0) bulk_wait_read<0>();  // the stores have read their blocks; the grid's end waits for the rest
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, BN);
  }
}

}  // namespace pomk

namespace pomh {

struct ClusterPlan {
  int bn, size;  // size 1: not by this kernel
};

// How many clusters of `size` CTAs run at once (clusters stay inside a group of SMs: 74 pairs, 33 fours, 15 eights here).
inline int max_clusters(int size) {
  static std::atomic<int> known[4];  // for 2, 4 and 8 at [1], [2], [3]; the devices of one machine are alike
  const int i = size == 2 ? 1 : size == 4 ? 2 : 3;
  int n = known[i].load(std::memory_order_relaxed);
  if (n) return n;
  auto kern = gemm_cluster_kernel<128, false>;
  constexpr int smem = ClusterSmem<128>::kBytes;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(64 * size));
  cfg.blockDim = dim3(kClusterThreads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = size, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) {
    (void)cudaGetLastError();
    return sm_count() / size * 3 / 4;  // no device to ask
  }
  known[i].store(n, std::memory_order_relaxed);
  return n;
}

// Estimated time in microseconds, launch apart: per wave of CTAs the k-blocks of one rank (0.285 each with 128 columns; 0.46 with
// 256, for which only three stages fit) and the exchange, which grows with the columns that a CTA finishes, against the same
// product by whole tiles.
inline ClusterPlan pick_cluster(int64_t M, int64_t N, int64_t K) {
  const int64_t kb = ceil_div(K, kBK), mt = ceil_div(M, kBM);
  const int sms = sm_count();
  // k-blocks of CTAs that take `bytes` each: bound by the SM's own intake, or by what the L2 gives all of them
  auto block_us = [](int64_t ctas, double alone, double bytes) {
    const double shared = static_cast<double>(ctas) * bytes / 13.5e6;
    return shared > alone ? shared : alone;
  };
  struct Whole {
    int64_t rows;
    int bn, slots, ctas;
    double alone, bytes;
  };
  const Whole whole[3] = {{mt, 128, sms, 1, 0.285, 32768.0}, {mt, 256, sms, 1, 0.37, 49152.0}, {(mt + 1) / 2, 256, sms / 2, 2, 0.335, 32768.0}};
  double best = -1.0;
  for (const Whole& w : whole) {
    const int64_t units = w.rows * ceil_div(N, w.bn), at_once = units < w.slots ? units : w.slots;
    const double t = ceil_div(units, w.slots) * (kb * block_us(at_once * w.ctas, w.alone, w.bytes) + 1.0);
    if (best < 0 || t < best) best = t;
  }
  best *= 0.97;  // an estimate this close is not worth the exchange
  ClusterPlan p{128, 1};
  for (int bn = 128; bn <= 256; bn += 128)
    for (int size = 2; size <= (bn == 128 ? kClusterMax : 2); size *= 2) {
      if (kb < 2 * size) continue;
      const int64_t units = mt * ceil_div(N, bn), slots = max_clusters(size), at_once = (units < slots ? units : slots) * size;
      const double block = bn == 128 ? block_us(at_once, 0.285, 32768.0) : block_us(at_once, 0.46, 49152.0);
      const double t = ceil_div(units, slots) * (ceil_div(kb, size) * block + 1.5 + 0.024 * (bn / size));
      if (t < best) best = t, p = ClusterPlan{bn, size};
    }
  return p;
}

template <int BN, bool B_MN>
int launch_cluster(const Operands& o, int size, ClusterDev d, int* status, cudaStream_t st) {
  CUtensorMap tmA, tmB, tmY, tmZ;
  int rc = build_maps(o, BN, &tmA, &tmB);
  if (rc) return rc;
  if ((rc = make_io_map(&tmY, d.y, o.N, o.M, 1, d.ldy))) return rc;
  tmZ = tmY;  // unused without z
  if (d.z && (rc = make_io_map(&tmZ, d.z, o.N, o.M, 1, o.N))) return rc;
  auto kern = gemm_cluster_kernel<BN, B_MN>;
  constexpr int smem = ClusterSmem<BN>::kBytes;
  static_assert(smem <= 232448, "more shared memory than a CTA may have");
  static std::atomic<uint64_t> attr_set{0};
  if ((rc = set_smem_once(kern, smem, &attr_set))) return rc;
  d.M = static_cast<int>(o.M), d.N = static_cast<int>(o.N);
  d.m_tiles = static_cast<int>(ceil_div(o.M, kBM));
  d.k_blocks = static_cast<int>(ceil_div(o.K, kBK));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(d.m_tiles * ceil_div(o.N, BN) * size));
  cfg.blockDim = dim3(kClusterThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = size, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, kern, tmA, tmB, tmY, tmZ, d, status) != cudaSuccess) {
    (void)cudaGetLastError();
    return POM_ERR_CUDA;
  }
  count_launch();
  return POM_OK;
}

// The product with the epilogue that `d` describes (its sizes are filled in here); K-major A, either B.
inline int cluster_product(const Operands& o, const ClusterPlan& p, ClusterDev d, int* status, cudaStream_t st) {
  const int rc = check_operands(o);
  if (rc) return rc;
  if (!d.has_bias) d.bias = o.A, d.bias_f32 = 0;
  if (!d.has_residual) d.residual = static_cast<const __nv_bfloat16*>(o.A), d.ldr = 0;
  if (o.b_mn)
    return p.bn == 128 ? launch_cluster<128, true>(o, p.size, d, status, st) : launch_cluster<256, true>(o, p.size, d, status, st);
  return p.bn == 128 ? launch_cluster<128, false>(o, p.size, d, status, st) : launch_cluster<256, false>(o, p.size, d, status, st);
}

}  // namespace pomh
