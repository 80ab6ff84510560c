// MXFP4 products on the block-scaled tensor-core kind: C [M, N] = A . B^T for
// A [M, K], B [N, K] in e2m1 codes with e8m0 scales (mxfp4.cu has the format).
//
// Per k-block of 256 elements a stage holds 128 bytes of each operand row
// (128-byte swizzle, as the 8- and 16-bit kernels) and the scale tiles of the
// same rows: two tiles of 512 bytes per 128 rows, copied to TMEM (tcgen05.cp)
// for the four MMAs (K = 64 each) of the k-block.
//
// An MMA is four times as short here as for 16-bit operands, so what bounds the
// product is how fast the k-blocks are issued (11136 x 28672 x 3584, one box):
//   one lane of one warp waits, copies scales and issues MMAs   646 us
//     (without the copies 460, one MMA of four 530; half the loads, fewer
//     stages or no stores: no change)
//   whole warps, a lane elected for the instructions            485 us
//     (without the copies 413, without waiting for a scale buffer 50 less)
//   scales copied by a warp of their own, one commit for both CTAs  415-425 us
//     (without the copies 373, one MMA of four 314, neither 306: operands
//     from L2 at 16 TB/s)
//
// Out-of-range rows, columns of K and scale tiles are filled with zeros by TMA:
// a zero code times 2^-127 is zero, so no tail needs a case of its own.
#pragma once

#include "tc_gemm.cuh"

namespace swiglu {

constexpr int kMxStageK = 256;           // elements of K per stage (128 bytes)
constexpr int kMxTileBytes = 512;        // one scale tile: 128 rows x 128 elements of K
constexpr int kMxScaleBytes = 2 * kMxTileBytes;  // of 128 rows per stage

// ------------------------------------------------------------ CTA pair, 256 x 256
struct MxParams {
  CUtensorMap tmA, tmB;    // codes, {128 bytes, 128 rows}
  CUtensorMap tmAs, tmBs;  // scale tiles as 32-bit cells, {256, 1}: both tiles of a stage
  CUtensorMap tmC;         // output, {32 x 32} boxes (SwiGLU: preact)
  CUtensorMap tmD;         // SwiGLU: h
  int M, N, K;
  int H, layout;           // SwiGLU: N = 2 H columns in `layout` order, H % 128 == 0
  bool store_preact, store_h;
  int tiles_m, tiles_n, group_m;
  uint32_t* status;
};

// TMEM: two 256-column accumulators that share 120 columns (0..255 and
// 136..391) leave 120 columns for scales, one buffer of 24 per stage of the
// ring, so that a stage's arrival also says that its scale buffer is free. The
// epilogue reads the shared columns first and frees them, then the next tile's
// MMAs may start: with two whole accumulators TMEM would be full.
// SWIGLU: a tile is the left and the gate columns of 128 hidden units, rank 0
// loading the left rows of B and rank 1 the gate rows, and the epilogue writes
// preact and h = left * silu(gate) (fused_forward.py:101-185).
template <bool OUT_F32_, bool SWIGLU_ = false>
struct MxCfg {
  static constexpr bool OUT_F32 = OUT_F32_;
  static constexpr bool SWIGLU = SWIGLU_;
  static constexpr int STAGES = 5;
  static constexpr int OPERAND_BYTES = 128 * 128;  // 128 rows
  static constexpr int SFA_OFFSET = 2 * OPERAND_BYTES;
  static constexpr int SFB_OFFSET = SFA_OFFSET + kMxScaleBytes;
  static constexpr int STAGE_BYTES = SFB_OFFSET + 2 * kMxScaleBytes;
  static constexpr int ACC_STEP = 136;             // accumulator 1 starts here
  static constexpr int SF_COL = ACC_STEP + 256;    // scale buffers, 24 columns a stage
  static constexpr int NUM_THREADS = 224;
  static constexpr int BAR_BYTES = 8 * (3 * STAGES + 5) + 16;
  static constexpr int EPI_OFFSET = STAGES * STAGE_BYTES + ((BAR_BYTES + 1023) / 1024) * 1024;
  static constexpr int EPI_WARP_BYTES = SWIGLU ? SwigluStage::kWarpBytes : StoreStage<OUT_F32>::kWarpBytes;
  static constexpr int SMEM_BYTES = 1024 + EPI_OFFSET + 4 * EPI_WARP_BYTES;
  static_assert(SF_COL + 24 * STAGES <= 512, "TMEM holds 512 columns");
  static_assert(STAGE_BYTES % 1024 == 0, "stages keep the swizzle's alignment");
  static_assert(SMEM_BYTES <= 227 * 1024, "shared memory budget");
};

// One {32 x 32} box of accumulator values to C through a swizzled staging
// buffer (StoreStage describes it).
template <bool OUT_F32>
__device__ __forceinline__ void mx_store_chunk(const CUtensorMap* map, const uint32_t (&r)[32], uint8_t* buf, int col,
                                               int row0) {
  using S = StoreStage<OUT_F32>;
  const uint32_t lane = threadIdx.x & 31u;
  if (lane == 0) bulk_wait_read<1>();  // the store issued from this buffer two boxes ago has read it
  __syncwarp();
  uint8_t* row_base = buf + lane * S::kRowBytes;
#pragma unroll
  for (int k = 0; k < S::kRowBytes / 16; ++k) {
    uint4 v;
    if constexpr (OUT_F32) {
      v = make_uint4(r[4 * k], r[4 * k + 1], r[4 * k + 2], r[4 * k + 3]);
    } else {
      v = make_uint4(pack_bf16x2(__uint_as_float(r[8 * k]), __uint_as_float(r[8 * k + 1])),
                     pack_bf16x2(__uint_as_float(r[8 * k + 2]), __uint_as_float(r[8 * k + 3])),
                     pack_bf16x2(__uint_as_float(r[8 * k + 4]), __uint_as_float(r[8 * k + 5])),
                     pack_bf16x2(__uint_as_float(r[8 * k + 6]), __uint_as_float(r[8 * k + 7])));
    }
    const int kk = OUT_F32 ? (k ^ static_cast<int>(lane & 7u)) : (k ^ static_cast<int>((lane >> 1) & 3u));
    *reinterpret_cast<uint4*>(row_base + 16 * kk) = v;
  }
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    tma_store_2d(map, buf, col, row0);
    bulk_commit();
  }
}

// One chunk of 32 hidden units of a SwiGLU tile: up to three {32 x 32} boxes
// (preact left, preact gate, h) through one staging area, as
// epilogue_swiglu_tma.
__device__ __forceinline__ void mx_swiglu_chunk(const MxParams& p, const uint32_t (&rl)[32], const uint32_t (&rg)[32],
                                                uint8_t* stage, int j, int row0) {
  const uint32_t lane = threadIdx.x & 31u;
  uint8_t* lbox = stage;
  uint8_t* gbox = stage + SwigluStage::kBoxBytes;
  uint8_t* hbox = stage + 2 * SwigluStage::kBoxBytes;
  if (lane == 0) bulk_wait_read<0>();  // the previous chunk's stores have read the boxes
  __syncwarp();
  float v[32];
  if (p.store_preact) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(rl[i]);
    stage_row32_bf16(lbox, lane, v);
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(rg[i]);
    stage_row32_bf16(gbox, lane, v);
  }
  if (p.store_h) {
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      // From the rounded preact, as the pointwise kernel of the other form; that one
      // has expf and a division in place of sigmoid_fast (as everywhere in this
      // library), so the last bit of a row's h may depend on the number of rows.
      const float l = bf16_round(__uint_as_float(rl[i])), g = bf16_round(__uint_as_float(rg[i]));
      v[i] = l * (g * sigmoid_fast(g));
    }
    stage_row32_bf16(hbox, lane, v);
  }
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    if (p.store_preact) {
      tma_store_2d(&p.tmC, lbox, left_col(j, p.H, p.layout), row0);
      tma_store_2d(&p.tmC, gbox, gate_col(j, p.H, p.layout), row0);
    }
    if (p.store_h) tma_store_2d(&p.tmD, hbox, j, row0);
    bulk_commit();
  }
}

template <class Cfg>
__global__ void __launch_bounds__(Cfg::NUM_THREADS, 1) mx_gemm_pair_kernel(const __grid_constant__ MxParams p) {
  wait_for_previous();
  constexpr int STAGES = Cfg::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + STAGES * Cfg::STAGE_BYTES);
  uint64_t* full = bars;                    // TMA (both CTAs) -> MMA; used in rank 0
  uint64_t* empty = bars + STAGES;          // MMA -> TMA, in each CTA
  uint64_t* scaled = bars + 2 * STAGES;     // scale copies -> MMA; used in rank 0
  uint64_t* tmem_full = bars + 3 * STAGES;  // MMA -> epilogue, in each CTA (2)
  uint64_t* tmem_free = tmem_full + 2;      // epilogues -> MMA; used in rank 0
  uint64_t* mma_done = tmem_free + 1;
  uint64_t* copies_done = mma_done + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(copies_done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const uint32_t warp = warp_id(), lane = lane_id();
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
      mbar_init(&scaled[s], 1);
    }
    for (int a = 0; a < 2; ++a) mbar_init(&tmem_full[a], 1);
    mbar_init(tmem_free, 8);
    mbar_init(mma_done, 1);
    mbar_init(copies_done, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before_sync();
  cluster_sync_all();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;

  const int num_kb = (p.K + kMxStageK - 1) / kMxStageK;
  const int tiles = p.tiles_m * p.tiles_n;
  const int first_tile = static_cast<int>(cluster_id_x());
  const int tile_step = static_cast<int>(num_clusters_x());
  uint32_t* status = p.status;

  if (warp == 0) {
    uint32_t stage = 0, phase = 0, filled = 0, fill_parity = 0;
    bool ok = true;
    for (int tile = first_tile; tile < tiles && ok; tile += tile_step) {
      int pm, pn;
      tile_coords(tile, p.tiles_m, p.tiles_n, p.group_m, pm, pn);
      const int am = 2 * pm + static_cast<int>(rank);  // 128-row tile of A of this CTA
      // 128-row tiles of B: the two halves of every MMA's columns.
      const int b0 = Cfg::SWIGLU ? left_col(pn * 128, p.H, p.layout) / 128 : 2 * pn;
      const int b1 = Cfg::SWIGLU ? gate_col(pn * 128, p.H, p.layout) / 128 : 2 * pn + 1;
      const int bn = leader ? b0 : b1;
      for (int kb = 0; kb < num_kb; ++kb) {
        if (!mbar_wait_warp(&empty[stage], phase ^ 1, abort_flag, status, kErrTimeoutProducer)) {
          ok = false;
          break;
        }
        if (elect_one()) {
          uint8_t* sa = smem + stage * Cfg::STAGE_BYTES;
          const uint32_t bar = map_to_rank(&full[stage], 0);
          if (leader) mbar_arrive_expect_tx(&full[stage], 2 * Cfg::STAGE_BYTES);
          tma_load_2d_pair(sa, &p.tmA, bar, kb * 128, am * 128);
          tma_load_2d_pair(sa + Cfg::OPERAND_BYTES, &p.tmB, bar, kb * 128, bn * 128);
          tma_load_2d_pair(sa + Cfg::SFA_OFFSET, &p.tmAs, bar, kb * 256, am);
          // Every MMA reads the scales of all 256 columns in both CTAs.
          tma_load_2d_pair(sa + Cfg::SFB_OFFSET, &p.tmBs, bar, kb * 256, b0);
          tma_load_2d_pair(sa + Cfg::SFB_OFFSET + kMxScaleBytes, &p.tmBs, bar, kb * 256, b1);
        }
        __syncwarp();
        filled |= 1u << stage;
        fill_parity = (fill_parity & ~(1u << stage)) | (phase << stage);
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    // Drain: a stage this CTA filled is finished once the MMA released it.
    for (int s = 0; s < STAGES; ++s) {
      if (filled & (1u << s)) {
        volatile int never = 0;
        mbar_wait_warp(&empty[s], (fill_parity >> s) & 1u, &never, status, kErrTimeoutTeardown);
      }
    }
  } else if (warp == 1) {
    if (leader) {
      constexpr uint32_t idesc[2] = {make_idesc_mxf4(256, 256, 0), make_idesc_mxf4(256, 256, 2)};
      const uint32_t smem0 = smem_u32(smem);
      uint32_t stage = 0, phase = 0, acc = 0, free_phase = 1;
      bool ok = true;
      for (int tile = first_tile; tile < tiles && ok; tile += tile_step) {
        // The previous tile's epilogue has read the columns both accumulators
        // share (and, before that, all of the tile before it).
        if (!mbar_wait_warp(tmem_free, free_phase, abort_flag, status, kErrTimeoutMma)) break;
        free_phase ^= 1;
        const uint32_t d_tmem = tmem_base + acc * Cfg::ACC_STEP;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait_warp(&scaled[stage], phase, abort_flag, status, kErrTimeoutMma)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t sa = smem0 + stage * Cfg::STAGE_BYTES;
          const uint32_t sb = sa + Cfg::OPERAND_BYTES;
          const uint32_t sfa = tmem_base + Cfg::SF_COL + 24 * stage, sfb = sfa + 8;
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              umma_mxf4_ss_pair(d_tmem, make_smem_desc_sw128(sa + k * 32, 16, 1024),
                                make_smem_desc_sw128(sb + k * 32, 16, 1024), idesc[k & 1], sfa + 4 * (k >> 1),
                                sfb + 8 * (k >> 1), (kb | k) != 0 ? 1u : 0u);
            }
            umma_commit_pair_both(&empty[stage]);
            if (kb + 1 == num_kb) umma_commit_pair_both(&tmem_full[acc]);
          }
          __syncwarp();
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
        acc ^= 1;
      }
      if (elect_one()) umma_commit_pair(map_to_rank(mma_done, 0));
      __syncwarp();
      volatile int never = 0;
      mbar_wait_warp(mma_done, 0, &never, status, kErrTimeoutTeardown);
    }
  } else if (warp == 6) {
    // Scale tiles of each stage to TMEM. The stage arrived, so its previous
    // MMAs, the last readers of its scale buffer, are done.
    if (leader) {
      const uint32_t smem0 = smem_u32(smem);
      uint32_t stage = 0, phase = 0;
      bool ok = true;
      for (int tile = first_tile; tile < tiles && ok; tile += tile_step) {
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait_warp(&full[stage], phase, abort_flag, status, kErrTimeoutMma)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t s = smem0 + stage * Cfg::STAGE_BYTES;
          const uint32_t sfa = tmem_base + Cfg::SF_COL + 24 * stage, sfb = sfa + 8;
          if (elect_one()) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              tmem_cp_scales_pair(sfa + 4 * t, make_smem_desc_scales(s + Cfg::SFA_OFFSET + t * kMxTileBytes));
#pragma unroll
              for (int h = 0; h < 2; ++h)
                tmem_cp_scales_pair(sfb + 8 * t + 4 * h,
                                    make_smem_desc_scales(s + Cfg::SFB_OFFSET + h * kMxScaleBytes + t * kMxTileBytes));
            }
            umma_commit_pair(map_to_rank(&scaled[stage], 0));
          }
          __syncwarp();
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      // The copies read shared memory and write TMEM: none outlives this warp.
      if (elect_one()) umma_commit_pair(map_to_rank(copies_done, 0));
      __syncwarp();
      volatile int never = 0;
      mbar_wait_warp(copies_done, 0, &never, status, kErrTimeoutTeardown);
    }
  } else {
    const uint32_t q = warp & 3u;
    uint32_t acc = 0, acc_phase = 0;
    uint8_t* stage = smem + Cfg::EPI_OFFSET + (warp - 2) * Cfg::EPI_WARP_BYTES;
    constexpr int kBufBytes = StoreStage<Cfg::OUT_F32>::kWarpBytes / 2;
    for (int tile = first_tile; tile < tiles; tile += tile_step) {
      int pm, pn;
      tile_coords(tile, p.tiles_m, p.tiles_n, p.group_m, pm, pn);
      if (!mbar_wait(&tmem_full[acc], acc_phase, abort_flag, status, kErrTimeoutEpilogue)) break;
      tc_fence_after_sync();
      const int row0 = pm * 256 + 128 * static_cast<int>(rank) + static_cast<int>(q * 32);
      const uint32_t t_row = tmem_base + ((q * 32u) << 16) + acc * Cfg::ACC_STEP;
      uint32_t r[4][32];
      auto free_shared = [&] {
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(map_to_rank(tmem_free, 0));
      };
      if constexpr (Cfg::SWIGLU) {
        // The shared columns are the gate half of accumulator 0 and the left half of
        // accumulator 1: one half is read and freed, the other follows chunk by chunk.
        const int half = acc == 0 ? 128 : 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_ld_32x32b_x32(t_row + half + i * 32, r[i]);
        tmem_ld_wait();
        free_shared();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t other[32];
          tmem_ld_32x32b_x32(t_row + (128 - half) + i * 32, other);
          tmem_ld_wait();
          if (acc == 0) mx_swiglu_chunk(p, other, r[i], stage, pn * 128 + i * 32, row0);
          else mx_swiglu_chunk(p, r[i], other, stage, pn * 128 + i * 32, row0);
        }
      } else {
        // Shared columns first: chunks 7..4 of accumulator 0, 0..3 of accumulator 1.
        const int c_first = acc == 0 ? 7 : 0, c_step = acc == 0 ? -1 : 1;
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_ld_32x32b_x32(t_row + (c_first + i * c_step) * 32, r[i]);
        tmem_ld_wait();
        free_shared();
#pragma unroll
        for (int i = 0; i < 4; ++i)
          mx_store_chunk<Cfg::OUT_F32>(&p.tmC, r[i], stage + (i & 1) * kBufBytes,
                                       pn * 256 + (c_first + i * c_step) * 32, row0);
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_ld_32x32b_x32(t_row + (c_first + (4 + i) * c_step) * 32, r[i]);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 4; ++i)
          mx_store_chunk<Cfg::OUT_F32>(&p.tmC, r[i], stage + (i & 1) * kBufBytes,
                                       pn * 256 + (c_first + (4 + i) * c_step) * 32, row0);
      }
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
    // The TMA stores read shared memory asynchronously: finish before exit.
    if (lane == 0) bulk_wait_read<0>();
  }

  // Neither CTA releases TMEM (or exits) before the pair is done with it.
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// ------------------------------------------------------------ clusters along K
// The kernel for outputs with too few 256 x 256 tiles to fill the device. The
// roles are swapped: the tensor core's 128-row operand is a tile of B (the
// weight), its columns are NT of A's M rows (the tokens; NT = 16..128), so with
// one token a weight byte is loaded once and nothing is padded but the columns.
// While the tiles are fewer than the CTAs that fit, a cluster of up to eight
// CTAs shares a tile and splits K; the parts are added in rank order through
// distributed shared memory, so no workspace is needed and results are
// run-to-run identical.
struct MxClusterParams {
  CUtensorMap tmW, tmWs;  // weight codes {128 bytes, 128 rows}, its scale tiles
  CUtensorMap tmX, tmXs;  // token codes {128 bytes, NT rows}, their scale tiles
  void* out;              // [M, N]
  int M, N, K;
  int tiles_x;            // token tiles
  uint32_t* status;
};

template <int NT_, bool OUT_F32_>
struct MxClusterCfg {
  static constexpr int NT = NT_;
  static constexpr bool OUT_F32 = OUT_F32_;
  static constexpr int W_BYTES = 128 * 128;
  static constexpr int X_BYTES = NT * 128;
  static constexpr int SFW_OFFSET = W_BYTES + X_BYTES;
  static constexpr int SFX_OFFSET = SFW_OFFSET + kMxScaleBytes;
  static constexpr int STAGE_BYTES = SFX_OFFSET + kMxScaleBytes;
  // About 105 KB a CTA, two CTAs an SM: twice what the latency of HBM asks for.
  static constexpr int STAGES = 107 * 1024 / STAGE_BYTES;
  static constexpr int SF_COL = NT;  // scale buffers: 16 columns each
  static constexpr int TMEM_COLS = NT + 32 <= 64 ? 64 : NT + 32 <= 128 ? 128 : 256;
  static constexpr int NUM_THREADS = 192;
  static constexpr int BAR_BYTES = 8 * (2 * STAGES + 1) + 16;
  static constexpr int SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + BAR_BYTES;
  static_assert(STAGES >= 2 && STAGES * STAGE_BYTES >= NT * 128 * 4, "the ring also holds the parts");
  static_assert(STAGE_BYTES % 1024 == 0, "stages keep the swizzle's alignment");
};

__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

template <class Cfg>
__global__ void __launch_bounds__(Cfg::NUM_THREADS) mx_gemm_cluster_kernel(const __grid_constant__ MxClusterParams p) {
  wait_for_previous();
  constexpr int STAGES = Cfg::STAGES, NT = Cfg::NT;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * Cfg::STAGE_BYTES);
  uint64_t* empty = full + STAGES;
  uint64_t* tmem_full = empty + STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tmem_full + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const uint32_t warp = warp_id(), lane = lane_id();
  const int rank = static_cast<int>(cluster_ctarank());
  const int parts = static_cast<int>(gridDim.x) / static_cast<int>(num_clusters_x());  // cluster size
  // Token tiles innermost: neighbours read the same weight tile.
  const int cluster = static_cast<int>(cluster_id_x());
  const int tile = cluster / p.tiles_x, x_tile = cluster % p.tiles_x;
  const int x0 = x_tile * NT, tokens = min(NT, p.M - x0);
  const int num_kb = (p.K + kMxStageK - 1) / kMxStageK;
  const int kb0 = rank * num_kb / parts, kb1 = (rank + 1) * num_kb / parts;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(tmem_full, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, Cfg::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  uint32_t* status = p.status;

  if (warp == 0) {
    uint32_t stage = 0, phase = 0, filled = 0, fill_parity = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!mbar_wait_warp(&empty[stage], phase ^ 1, abort_flag, status, kErrTimeoutProducer)) break;
      if (elect_one()) {
        uint8_t* s = smem + stage * Cfg::STAGE_BYTES;
        mbar_arrive_expect_tx(&full[stage], Cfg::STAGE_BYTES);
        tma_load_2d(s, &p.tmW, &full[stage], kb * 128, tile * 128);
        tma_load_2d(s + Cfg::SFW_OFFSET, &p.tmWs, &full[stage], kb * 256, tile);
        tma_load_2d(s + Cfg::W_BYTES, &p.tmX, &full[stage], kb * 128, x0);
        tma_load_2d(s + Cfg::SFX_OFFSET, &p.tmXs, &full[stage], kb * 256, x0 / 128);
      }
      __syncwarp();
      filled |= 1u << stage;
      fill_parity = (fill_parity & ~(1u << stage)) | (phase << stage);
      if (++stage == STAGES) {
        stage = 0;
        phase ^= 1;
      }
    }
    // Drain: every load this warp issued must land before the CTA exits.
    for (int s = 0; s < STAGES; ++s) {
      if (filled & (1u << s)) {
        volatile int never = 0;
        mbar_wait_warp(&full[s], (fill_parity >> s) & 1u, &never, status, kErrTimeoutTeardown);
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc[2] = {make_idesc_mxf4(128, NT, 0), make_idesc_mxf4(128, NT, 2)};
    uint32_t stage = 0, phase = 0, old_stage = 0, old_phase = 0, sf = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!mbar_wait_warp(&full[stage], phase, abort_flag, status, kErrTimeoutMma)) break;
      if (kb >= kb0 + 2) {  // the MMAs that read this scale buffer last
        if (!mbar_wait_warp(&empty[old_stage], old_phase, abort_flag, status, kErrTimeoutMma)) break;
        if (++old_stage == STAGES) {
          old_stage = 0;
          old_phase ^= 1;
        }
      }
      tc_fence_after_sync();
      const uint32_t sw = smem_u32(smem + stage * Cfg::STAGE_BYTES), sx = sw + Cfg::W_BYTES;
      const uint32_t sfw = tmem_base + Cfg::SF_COL + 16 * sf, sfx = sfw + 8;
      if (elect_one()) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          tmem_cp_scales(sfw + 4 * t, make_smem_desc_scales(sw + Cfg::SFW_OFFSET + t * kMxTileBytes));
          tmem_cp_scales(sfx + 4 * t, make_smem_desc_scales(sw + Cfg::SFX_OFFSET + t * kMxTileBytes));
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          umma_mxf4_ss(tmem_base, make_smem_desc_sw128(sw + k * 32, 16, 1024),
                       make_smem_desc_sw128(sx + k * 32, 16, 1024), idesc[k & 1], sfw + 4 * (k >> 1),
                       sfx + 4 * (k >> 1), (kb != kb0 || k != 0) ? 1u : 0u);
        }
        umma_commit(&empty[stage]);
      }
      __syncwarp();
      sf ^= 1;
      if (++stage == STAGES) {
        stage = 0;
        phase ^= 1;
      }
    }
    if (elect_one()) umma_commit(tmem_full);  // arrives when all MMAs issued so far are done
    __syncwarp();
    volatile int never = 0;
    mbar_wait_warp(tmem_full, 0, &never, status, kErrTimeoutTeardown);
  }

  // Each CTA lays its part down as [token][weight row] over the ring (its MMAs
  // are done), then the CTAs of the cluster share the tokens: a thread adds four
  // neighbouring rows of a token over the parts, in rank order, and stores them.
  float* part = reinterpret_cast<float*>(smem);
  bool ok = true;
  if (warp >= 2) {
    ok = mbar_wait(tmem_full, 0, abort_flag, status, kErrTimeoutEpilogue);
    if (ok) {
      tc_fence_after_sync();
      const uint32_t q = warp & 3u;
      const int row = static_cast<int>(q * 32 + lane);  // TMEM lane = weight row
#pragma unroll 1
      for (int c = 0; c < tokens; c += 16) {
        uint32_t r[16];
        tmem_ld_32x32b_x16(tmem_base + ((q * 32u) << 16) + c, r);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) part[(c + i) * 128 + row] = __uint_as_float(r[i]);
      }
    }
  }
  if (parts > 1) cluster_sync_all();
  else if (warp >= 2) asm volatile("bar.sync 1, 128;" ::: "memory");
  const int n = tile * 128 + static_cast<int>(lane) * 4;
  if (warp >= 2 && ok && n < p.N) {  // N is a multiple of 8: groups of four are whole
    const uint32_t mine = smem_u32(part) + lane * 16;
#pragma unroll 4
    for (int t = rank + static_cast<int>(warp - 2) * parts; t < tokens; t += 4 * parts) {
      float4 v[8];
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        if (s < parts) v[s] = ld_cluster_f32x4(map_to_rank(mine + t * 512, s));
      }
#pragma unroll
      for (int s = 1; s < 8; ++s) {
        if (s < parts) v[0] = make_float4(v[0].x + v[s].x, v[0].y + v[s].y, v[0].z + v[s].z, v[0].w + v[s].w);
      }
      const long long at = static_cast<long long>(x0 + t) * p.N + n;
      if constexpr (Cfg::OUT_F32) {
        *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = v[0];
      } else {
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + at) =
            make_uint2(pack_bf16x2(v[0].x, v[0].y), pack_bf16x2(v[0].z, v[0].w));
      }
    }
  }
  if (parts > 1) cluster_sync_all();  // no CTA leaves while another reads its part

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
  }
}

}  // namespace swiglu
