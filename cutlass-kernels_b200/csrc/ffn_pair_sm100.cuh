// The feed-forward products on CTA pairs: tiles of 256 rows x up to 256 columns of accumulator, as in gemm_sm100.cu, for operands and
// results that a plain GEMM does not have.
//
//   kProductI8   8-bit integers (kind::i8, 128 elements per 128-byte k-block, int32 sums), scaled per row and column at the end
//   kGated16/I8  the leader's half of the accumulator columns is the gate projection and its peer's half the up projection: each
//                CTA loads rows of ONE of the two weights, so the pair's accumulator holds gate and up of the same columns
//                of h, and the epilogue has both of an element in one thread.  x is read once for the two products.
//   kGrad        two lists of tiles in one launch, the longer tiles first.  dx: one reduction over the channels of w_gate and then of
//                w_up, so it leaves the tensor core summed; the weights are stored with the model's width contiguous, which
//                is the column of dx: they are MN-major operands.  dw_gate, dw_up: a reduction over the tokens, along which neither
//                operand is contiguous: both are MN-major.
//
// Roles, ring, tensor-memory double buffer and store path are those of gemm_kernel: warp 0 TMA, warp 1 of the leader
// UMMA (cta_group::2), but two groups of four epilogue warps (with one, a tile's epilogue of 3 us was most of a short call) that store
// with TMA, which clips at the result's edges.
// An MN-major operand lands as spans of 64 columns, [span][64 k-rows][128 bytes], each with the 128-byte swizzle; what lies
// behind a matrix is zero-filled in both operands, so ragged reductions need no mask.
//
// A tile is 2 bn accumulator columns wide, bn = 128, 96 or 64 by what fills the last wave of pairs best (ffn.cu).  Bound by the tensor
// core: 512 clk of MMA per k-block of 128 bytes at bn = 128 against 32 KB of loads per SM and, in the gated modes, an epilogue of
// two special-function operations per element of h that runs beside the next tile's main loop.
#pragma once
#include "common.cuh"
#include "ffn_act.cuh"
#include "ffn_params.h"
#include "gemm_tiles.cuh"
#include "host_util.h"

namespace cfk {

constexpr int kErrPairFull = 211, kErrPairEmpty = 212, kErrPairAccFull = 213, kErrPairAccEmpty = 214, kErrPairStaged = 215,
              kErrPairStageFree = 216;

struct PairCfg {
  static constexpr int TM = 256, TN = 256, BM = 128, BN = 128;     // tile of the pair; rows of X and of Y per CTA
  static constexpr int XB = BM * 128, YB = BN * 128;               // bytes per k-block
  static constexpr int NSTAGE = 6;
  static constexpr int GROUPS = 2;                                 // of four epilogue warps
  static constexpr int STAGEB = 128 * 128;                         // staging per group: 128 rows x 32 columns of fp32, or twice 16 bits
  static constexpr int SMEM_BYTES = 1024 + NSTAGE * (XB + YB) + GROUPS * STAGEB + 256;
  static constexpr int NTHREADS = 64 + GROUPS * 128;
  static_assert(8 * (2 * NSTAGE + 4 + 4 * GROUPS) + 8 <= 256, "barrier block overflows");
};

// 32 columns of 128 rows as a TMA store takes them: rows of 64 bytes with the 64-byte swizzle (16-byte piece index XOR bits 1-2 of
// the row), or of 128 bytes with the 128-byte swizzle (XOR bits 0-2) for fp32.
__device__ __forceinline__ uint32_t staged_at(uint32_t tile, int r, uint32_t byte, bool out32) {
  return out32 ? tile + r * 128 + (((byte >> 4) ^ (uint32_t)(r & 7)) << 4) + (byte & 15u)
               : tile + r * 64 + (((byte >> 4) ^ (uint32_t)((r >> 1) & 3)) << 4) + (byte & 15u);
}
__device__ __forceinline__ void stage_row16(uint32_t tile, int r, bool bf16, const float (&v)[32]) {
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const uint32_t w0 = pack_out(bf16, v[g * 8], v[g * 8 + 1]), w1 = pack_out(bf16, v[g * 8 + 2], v[g * 8 + 3]);
    const uint32_t w2 = pack_out(bf16, v[g * 8 + 4], v[g * 8 + 5]), w3 = pack_out(bf16, v[g * 8 + 6], v[g * 8 + 7]);
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(staged_at(tile, r, g * 16, false)), "r"(w0), "r"(w1), "r"(w2),
                 "r"(w3) : "memory");
  }
}
__device__ __forceinline__ void stage_row32(uint32_t tile, int r, const float (&v)[32]) {
#pragma unroll
  for (int g = 0; g < 8; ++g)
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(staged_at(tile, r, g * 16, true)),
                 "r"(__float_as_uint(v[g * 4])), "r"(__float_as_uint(v[g * 4 + 1])), "r"(__float_as_uint(v[g * 4 + 2])),
                 "r"(__float_as_uint(v[g * 4 + 3])) : "memory");
}

// A TMA store writes whole 16-byte pieces: behind the last element of a row it would put zeros up to the next multiple of 16
// bytes.  So the descriptors of the results end at the last whole piece, column `whole`, and the columns from there on are
// stored one by one, read back from this thread's own row of the staged 32 columns that begin at `col`.
__device__ __forceinline__ int whole_columns(int cols, bool out32) { return cols & ~(out32 ? 3 : 7); }
__device__ __forceinline__ void store_rest(const ProductParams& p, int which, bool out32, uint32_t tile, int r, int row, int col,
                                           int whole, int cols) {
  const int end = cols < col + 32 ? cols : col + 32;
  for (int c = whole > col ? whole : col; c < end; ++c) {
    const uint32_t from = staged_at(tile, r, (uint32_t)((c - col) * (out32 ? 4 : 2)), out32);
    const int64_t at = row * p.d_stride[which] + c;
    if (out32) {
      uint32_t v;
      asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(from) : "memory");
      reinterpret_cast<uint32_t*>(p.d[which])[at] = v;
    } else {
      uint16_t v;
      asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(from) : "memory");
      reinterpret_cast<uint16_t*>(p.d[which])[at] = v;
    }
  }
}

// h = act(gate) * up in place of gate
template <int ACT>
__device__ __forceinline__ void gate_by(float (&gate)[32], const float (&up)[32]) {
#pragma unroll
  for (int i = 0; i < 32; ++i) gate[i] = activate<ACT>(gate[i]) * up[i];
}
__device__ __forceinline__ void gate_columns(int act, float (&gate)[32], const float (&up)[32]) {
  switch (act) {
    case CFK_ACT_SILU: gate_by<CFK_ACT_SILU>(gate, up); break;
    case CFK_ACT_GELU: gate_by<CFK_ACT_GELU>(gate, up); break;
    case CFK_ACT_GELU_TANH: gate_by<CFK_ACT_GELU_TANH>(gate, up); break;
    default: gate_by<CFK_ACT_RELU>(gate, up); break;
  }
}

// A tile of the launch: its list, its place and its reduction.
struct PairTile {
  int kind, tr, tc, batch, bn, rows, cols, nkb_part, nkb;
};
// The `local`-th tile of a pair; false: it has no more (see PairPlan for the order).
__device__ __forceinline__ bool pair_tile(PairTile& t, const PairPlan& plan, int pair, int local, bool grad, int kb) {
  const int first = plan.job[0].tiles_r * plan.job[0].tiles_c * plan.job[0].batches, pairs = plan.pairs;
  const int mine = first > pair ? (first - pair + pairs - 1) / pairs : 0;
  int j = 0, tile = pair + local * pairs;
  if (local >= mine) {
    if (plan.jobs < 2) return false;
    const int i = local - mine, more = first % pairs;
    j = 1;
    tile = pair < more ? i * more + pair : more * plan.share + i * (pairs - more) + (pair - more);
    if (pair < more ? i >= plan.share : tile >= plan.job[1].tiles_r * plan.job[1].tiles_c * plan.job[1].batches) return false;
  }
  const PairJob& job = plan.job[j];
  t.kind = job.kind; t.bn = job.bn; t.rows = job.rows; t.cols = job.cols;
  tile_coords(tile, job.tiles_r, job.tiles_c, t.tr, t.tc, t.batch);
  t.nkb_part = (job.reduce + kb - 1) / kb;
  t.nkb = grad && t.kind == 0 ? 2 * t.nkb_part : t.nkb_part;
  return true;
}

template <int MODE>
__global__ void __launch_bounds__(PairCfg::NTHREADS, 1)
pair_product_kernel(const __grid_constant__ ProductMaps maps, const __grid_constant__ ProductParams p,
                    const __grid_constant__ PairPlan plan) {
  using C = PairCfg;
  constexpr bool I8 = MODE == kProductI8 || MODE == kGatedI8;
  constexpr bool GATED = MODE == kGated16 || MODE == kGatedI8;
  constexpr bool GRAD = MODE == kGrad;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t sX = smem_base;
  const uint32_t sY = smem_base + C::NSTAGE * C::XB;
  const uint32_t sStage = sY + C::NSTAGE * C::YB;            // [GROUPS] output staging
  const uint32_t sBar = sStage + C::GROUPS * C::STAGEB;
  const uint32_t bar_full = sBar;                            // [NSTAGE] leader: both CTAs' loads of a stage landed
  const uint32_t bar_empty = sBar + 8 * C::NSTAGE;           // [NSTAGE] each CTA: its stage was consumed
  const uint32_t bar_acc_full = bar_empty + 8 * C::NSTAGE;   // [2] each CTA: accumulator complete
  const uint32_t bar_acc_empty = bar_acc_full + 16;          // [2] leader: all epilogue warps of both have read it
  const uint32_t bar_staged = bar_acc_empty + 16;            // [GROUPS][2] a staging tile is complete (4 epilogue warps)
  const uint32_t bar_stage_free = bar_staged + 16 * C::GROUPS;   // [GROUPS][2] the TMA store has read a staging tile
  uint8_t* gBar = smem_gen + (sBar - smem_base);
  const uint32_t off_misc = 8 * (2 * C::NSTAGE + 4 + 4 * C::GROUPS);
  volatile uint32_t* s_tmem_base = reinterpret_cast<volatile uint32_t*>(gBar + off_misc);
  volatile uint32_t* s_abort = reinterpret_cast<volatile uint32_t*>(gBar + off_misc + 4);
  const AbortCtx actx{s_abort, p.status};

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_ctarank();                   // 0 = leader
  const int pair_id = (int)(blockIdx.x >> 1);
  constexpr int KB = I8 ? 128 : 64;                          // elements of the reduction per k-block

  cluster_arrive_started();
  if (tid == 0) {
    for (int i = 0; i < C::NSTAGE; ++i) { mbar_init(bar_full + 8 * i, 2); mbar_init(bar_empty + 8 * i, 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(bar_acc_full + 8 * i, 1); mbar_init(bar_acc_empty + 8 * i, 2 * 4 * C::GROUPS); }
    for (int i = 0; i < 2 * C::GROUPS; ++i) { mbar_init(bar_staged + 8 * i, 4); mbar_init(bar_stage_free + 8 * i, 1); }
    *s_abort = 0u;
    fence_barrier_init();
  }
  __syncwarp();
  cluster_wait_started();
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(const_cast<uint32_t*>(s_tmem_base)), 2 * C::TN);
    tmem_relinquish_pair();
    grid_dependency_launch();
  }
  if (warp == 0 && lane == 0) { tma_prefetch_desc(&maps.x[0]); tma_prefetch_desc(&maps.y[0]); }
  grid_dependency_wait();
  tc_fence_before_sync();
  const bool skip = pair_should_skip(p.status);              // one decision for the pair
  tc_fence_after_sync();
  const uint32_t tmem_base = *s_tmem_base;
  if (skip) {
    if (warp == 1) tmem_dealloc_pair(tmem_base, 2 * C::TN);
    return;
  }

  if (warp == 0) {
    if (lane == 0) {
      int idx = 0, local = 0;
      bool ok = true;
      for (PairTile t; ok && pair_tile(t, plan, pair_id, local, GRAD, KB); ++local) {
        const int xr = t.tr * C::TM + (int)rank * C::BM;                                    // first of this CTA's rows of X
        const int yr = GATED ? t.tc * t.bn : t.tc * 2 * t.bn + (int)rank * t.bn;            // and of Y
        const uint32_t bytes = C::XB + (GRAD ? (t.bn > 64 ? C::YB : C::YB / 2) : t.bn * 128);
        for (int i = 0; i < t.nkb; ++i, ++idx) {
          // every other tile walks the reduction backwards, from the k-blocks that are still in L2 (gemm_sm100.cu)
          const int kb = (local & 1) ? t.nkb - 1 - i : i;
          const int part = GRAD && kb >= t.nkb_part ? 1 : 0;
          const int k = (kb - part * t.nkb_part) * KB;
          const int s = idx % C::NSTAGE;
          const uint32_t ph = (idx / C::NSTAGE) & 1;
          if (!mbar_wait(bar_empty + 8 * s, ph ^ 1u, actx, kErrPairEmpty)) { ok = false; break; }
          const uint32_t full = map_to_cta(bar_full + 8 * s, 0);
          const uint32_t x = sX + s * C::XB, y = sY + s * C::YB;
          mbar_arrive_expect_tx_cluster(full, bytes);
          if constexpr (GRAD) {      // boxes of 64 x 64
            const CUtensorMap* mx = &maps.x[t.kind == 0 ? part : t.batch];
            const CUtensorMap* my = &maps.y[t.kind == 0 ? part : 2];
            tma_load_3d_pair(x, mx, full, t.kind == 0 ? k : xr, t.kind == 0 ? xr : k, 0);
            tma_load_3d_pair(x + C::XB / 2, mx, full, t.kind == 0 ? k : xr + 64, t.kind == 0 ? xr + 64 : k, 0);
            tma_load_3d_pair(y, my, full, yr, k, 0);
            if (t.bn > 64) tma_load_3d_pair(y + C::YB / 2, my, full, yr + 64, k, 0);
          } else {
            tma_load_3d_pair(x, &maps.x[0], full, k, xr, 0);
            tma_load_3d_pair(y, &maps.y[GATED ? (int)rank : 0], full, k, yr, 0);
          }
        }
      }
    }
  } else if (warp == 1) {
    // UMMA issue: all 32 lanes of the leader's warp run the loop, one elected lane executes the instructions
    if (rank == 0) {
      const uint32_t leader = elect_one();
      const uint32_t fmt = p.bf16 ? kFmtBF16 : kFmtF16;
      int idx = 0, local = 0;
      bool ok = true;
      for (PairTile t; ok && pair_tile(t, plan, pair_id, local, GRAD, KB); ++local) {
        const bool x_mn = GRAD && t.kind == 1;
        const uint32_t idesc = I8 ? make_idesc(2, kFmtS8, kFmtS8, 0, 0, C::TM, 2 * t.bn)
                                  : make_idesc(1, fmt, fmt, x_mn ? 1 : 0, GRAD ? 1 : 0, C::TM, 2 * t.bn);
        // 32 bytes along the reduction, or 16 rows of 128 bytes, per instruction
        const uint32_t xstep = x_mn ? 2048 : 32, xlbo = x_mn ? C::XB / 2 : 16;
        constexpr uint32_t YSTEP = GRAD ? 2048 : 32, YLBO = GRAD ? C::YB / 2 : 16;
        const int buf = local & 1;
        if (!mbar_wait_warp(bar_acc_empty + 8 * buf, ((local >> 1) & 1) ^ 1u, actx, kErrPairAccEmpty)) { ok = false; break; }
        tc_fence_after_sync();
        const uint32_t d = tmem_base + buf * C::TN;
        for (int i = 0; i < t.nkb; ++i, ++idx) {
          const int s = idx % C::NSTAGE;
          if (!mbar_wait_warp(bar_full + 8 * s, (idx / C::NSTAGE) & 1, actx, kErrPairFull)) { ok = false; break; }
          tc_fence_after_sync();
          const uint64_t a0 = make_smem_desc(sX + s * C::XB, xlbo, 1024, kSwizzle128B);
          const uint64_t b0 = make_smem_desc(sY + s * C::YB, YLBO, 1024, kSwizzle128B);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            const uint64_t a = desc_advance(a0, kk * xstep), bd = desc_advance(b0, kk * YSTEP);
            if constexpr (I8) umma_ss_i8<true>(d, a, bd, idesc, (i | kk) != 0 ? 1u : 0u, leader);
            else umma_ss_e<false, true>(d, a, bd, idesc, (i | kk) != 0 ? 1u : 0u, leader);
          }
          umma_commit_pair_e(bar_empty + 8 * s, (uint16_t)3, leader);      // the stage is free in both CTAs
        }
        if (ok) umma_commit_pair_e(bar_acc_full + 8 * buf, (uint16_t)3, leader);
      }
    }
  } else {
    // epilogue warps 2..9 in two groups of four; warp w may touch TMEM lanes 32*(w%4) .. +31.  A tile leaves in chunks of 32 columns,
    // taken by the groups in turn, each through staging of the group's own (two tiles that alternate; one of fp32).  With `keep`
    // the chunks of h, gate and up of the same columns follow each other.
    const int grp = (warp - 2) >> 2;
    const int q = warp & 3;
    const int r = q * 32 + lane;                       // row within this CTA's 128 rows
    const uint32_t lane_base = (uint32_t)(q * 32) << 16;
    const uint32_t leader_acc_empty = map_to_cta(bar_acc_empty, 0);
    const uint32_t my_stage = sStage + grp * C::STAGEB, my_staged = bar_staged + 16 * grp, my_free = bar_stage_free + 16 * grp;
    const bool out32 = MODE == kProductI8 && p.out == CFK_FP32, out_bf16 = p.out == CFK_BF16;
    const int kinds = GATED && p.keep ? 3 : 1;         // chunks per 32 columns: h, gate, up
    const bool storer = ((warp - 2) & 3) == 0 && lane == 0;
    int local = 0;
    uint32_t n = 0;                                    // chunks this group has staged so far
    bool ok = true;
    for (PairTile t; ok && pair_tile(t, plan, pair_id, local, GRAD, KB); ++local) {
      const int buf = local & 1;
      const int row0 = t.tr * C::TM + (int)rank * C::BM, row = row0 + r;
      const int tcols = GATED ? t.bn : 2 * t.bn, col0 = t.tc * tcols;
      const int end = t.cols - col0 < tcols ? t.cols - col0 : tcols;     // columns of the tile that exist
      const int whole = whole_columns(t.cols, out32);
      const uint32_t acc = tmem_base + lane_base + buf * C::TN;
      float rs = 0.f;
      if constexpr (I8) rs = row < t.rows ? __ldg(p.row_scale + row) : 0.f;
      ok = mbar_wait_warp(bar_acc_full + 8 * buf, (local >> 1) & 1, actx, kErrPairAccFull);
      if (!ok) break;
      tc_fence_after_sync();
      const int nchunk = (end + 31) / 32 * kinds;
#pragma unroll 1
      for (int ch = grp; ch < nchunk; ch += C::GROUPS, ++n) {
        const int kind = kinds == 1 ? 0 : ch % 3;
        const int which = GRAD ? (t.kind == 0 ? 0 : 1 + t.batch) : kind;   // result
        const int cb = (kinds == 1 ? ch : ch / 3) * 32;                    // first column of the chunk within the tile
        const uint32_t sb = out32 ? 0u : n & 1u, use = out32 ? n : n >> 1; // staging tile and how often it was used before
        const uint32_t stage = my_stage + sb * (C::STAGEB / 2);
        if (use >= 1u) {   // the store that last used this staging tile has read it
          ok = mbar_wait_warp(my_free + 8 * sb, (use & 1u) ^ 1u, actx, kErrPairStageFree);
          if (!ok) break;
        }
        const int col = col0 + cb + lane;                      // this lane's column: its scales reach the others by shuffle
        float v[32];
        if constexpr (GATED) {
          float gs = 1.f, us = 1.f;
          if constexpr (I8) {
            gs = col < t.cols ? __ldg(p.col_scale + col) : 0.f;
            us = col < t.cols ? __ldg(p.col_scale2 + col) : 0.f;
          }
          float u[32];
          uint32_t w[32];
          if (kind != 2) {
            tmem_ld_x32(acc + cb, w);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              if constexpr (I8) v[i] = __int2float_rn((int)w[i]) * rs * __shfl_sync(0xffffffffu, gs, i);
              else v[i] = __uint_as_float(w[i]);
            }
          }
          if (kind != 1) {
            tmem_ld_x32(acc + t.bn + cb, w);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              if constexpr (I8) u[i] = __int2float_rn((int)w[i]) * rs * __shfl_sync(0xffffffffu, us, i);
              else u[i] = __uint_as_float(w[i]);
            }
          }
          if (kind == 0) gate_columns(p.act, v, u);
          if (kind == 2) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = u[i];
          }
          stage_row16(stage, r, out_bf16, v);
        } else {
          uint32_t w[32];
          tmem_ld_x32(acc + cb, w);
          tmem_wait_ld();
          if constexpr (I8) {
            const float cs = col < t.cols ? __ldg(p.col_scale + col) : 0.f;
            const float bs = p.bias != nullptr && col < t.cols ? __ldg(p.bias + col) : 0.f;
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __int2float_rn((int)w[i]) * rs * __shfl_sync(0xffffffffu, cs, i);
            if (p.bias != nullptr) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] += __shfl_sync(0xffffffffu, bs, i);
            }
            if (out32) stage_row32(stage, r, v);
            else stage_row16(stage, r, out_bf16, v);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(w[i]);
            stage_row16(stage, r, out_bf16, v);
          }
        }
        if (row < t.rows && col0 + cb + 32 > whole) store_rest(p, which, out32, stage, r, row, col0 + cb, whole, t.cols);
        fence_proxy_async_smem();
        mbar_arrive_warp(my_staged + 8 * sb);
        if (storer) {
          if (!mbar_wait(my_staged + 8 * sb, use & 1u, actx, kErrPairStaged)) { ok = false; }
          else {
            if (col0 + cb < whole) tma_store_3d(&maps.d[which], stage, col0 + cb, row0, 0);
            tma_store_commit();
            if (out32) {
              tma_store_wait_read0();
              mbar_arrive(my_free);
            } else {
              tma_store_wait_read1();          // every store but this one has read its staging tile
              if (n >= 1u) mbar_arrive(my_free + 8 * (sb ^ 1u));
            }
          }
        }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
      }
      // this warp has read the accumulator: the next tile but one may overwrite it
      tc_fence_before_sync();
      if (ok) mbar_arrive_cluster_warp(leader_acc_empty + 8 * buf);
    }
    if (storer) tma_store_wait_read0();
  }

  settle_if_aborted(s_abort);
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();           // no CTA leaves while its peer may still signal it
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, 2 * C::TN);
  }
}

template <int MODE>
int launch_pair_product(const ProductMaps& maps, const ProductParams& p, const PairPlan& plan, cudaStream_t stream) {
  using C = PairCfg;
  static thread_local int attr_dev = -1;
  int dev = 0;
  if (note_cuda(cudaGetDevice(&dev), "cudaGetDevice") != cudaSuccess) return CFK_ERR_NO_DRIVER;
  if (attr_dev != dev) {
    if (note_cuda(cudaFuncSetAttribute(pair_product_kernel<MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES),
                  "cudaFuncSetAttribute(product smem)") != cudaSuccess)
      return CFK_ERR_LAUNCH;
    attr_dev = dev;
  }
  return note_cuda(launch_overlapped_in(2, pair_product_kernel<MODE>, dim3((unsigned)(2 * plan.pairs)), dim3(C::NTHREADS),
                                        C::SMEM_BYTES, stream, maps, p, plan), "product launch") == cudaSuccess ? CFK_OK
                                                                                                                : CFK_ERR_LAUNCH;
}

}  // namespace cfk
