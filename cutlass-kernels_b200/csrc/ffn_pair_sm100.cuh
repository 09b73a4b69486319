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
// Roles, ring and tensor-memory double buffer are those of gemm_kernel: warp 0 TMA, warp 1 of the leader UMMA (cta_group::2); but
// two groups of four epilogue warps, which write with ordinary stores.  (A TMA store writes whole 16-byte pieces, so behind the
// last element of a row it would put zeros up to the next multiple of 16 bytes; and the hand-over of staging tiles between four
// warps and a storing thread took 0.6 us per 32 columns, most of a tile whose reduction is short.)
// An MN-major operand lands as spans of 64 columns, [span][64 k-rows][128 bytes], each with the 128-byte swizzle; what lies
// behind a matrix is zero-filled in both operands, so ragged reductions need no mask.
//
// A tile is 2 bn accumulator columns wide, bn = 128, 96 or 64 by what fills the last wave of pairs best (ffn.cu).  Bound by the tensor
// core: 512 clk of MMA per k-block of 128 bytes at bn = 128 against 32 KB of loads per SM and, in the gated modes, an epilogue of
// two special-function operations per element of h that runs beside the next tile's main loop.  The pipe is 88 to 96 % active, at
// the 1.15 to 1.3 GHz that the power cap leaves, and the range between boxes is wide: gated 8192 x 11264 x 4096 in bf16 1051 to 1121 us, 1350
// to 1440 TFLOP/s; its 8-bit form 507 to 553 us; 8192^3 in 8 bits 334 us (3290 TOP/s) for a few launches and 370 to 413 (2660 to 2970) for
// seconds on end; the gradients of 8192 x 11264 x 4096 2300 to 2790 us, 1080 to 1310 TFLOP/s.
#pragma once
#include <type_traits>

#include "common.cuh"
#include "ffn_act.cuh"
#include "ffn_params.h"
#include "gemm_tiles.cuh"
#include "host_util.h"

namespace cfk {

constexpr int kErrPairFull = 211, kErrPairEmpty = 212, kErrPairAccFull = 213, kErrPairAccEmpty = 214;

struct PairCfg {
  static constexpr int TM = 256, TN = 256, BM = 128, BN = 128;     // tile of the pair; rows of X and of Y per CTA
  static constexpr int XB = BM * 128, SPANB = 64 * 128;            // bytes per k-block: of X; of a 64 x 64 box of an MN-major operand
  static constexpr int GROUPS = 2;                                 // of four epilogue warps
  static constexpr int HEADB = 1024 + 256, MAXSTAGE = 8;           // alignment slack and the barrier block
  static constexpr int STAGEB = 32 * 128;                          // output staging of an epilogue warp, where results are staged
  static constexpr int NTHREADS = 64 + GROUPS * 128;
  static constexpr int SMEM = 227 * 1024 - 128;                    // and a few static bytes of the kernel
  static_assert(8 * (2 * MAXSTAGE + 4) + 8 <= 256, "barrier block overflows");
};

// Results leave in one of two ways.
// From registers: a thread has a row and writes 32 columns of it, in whole 32-byte sectors where rows start at multiples of 32 bytes
// (`wide`), and nothing behind the row's end.
__device__ __forceinline__ void st_global_32(void* to, const uint32_t (&w)[32], int at) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[at]), "r"(w[at + 1]), "r"(w[at + 2]),
               "r"(w[at + 3]), "r"(w[at + 4]), "r"(w[at + 5]), "r"(w[at + 6]), "r"(w[at + 7]) : "memory");
}
__device__ __forceinline__ void store_columns(const ProductParams& p, int which, int row, int col, int cols, const float (&v)[32]) {
  const bool out32 = p.out == CFK_FP32, bf16 = p.out == CFK_BF16;
  const int64_t at = row * p.d_stride[which] + col;
  const int n = cols - col;                      // columns that exist, if fewer than 32
  uint32_t w[32];
  if (out32) {
    float* d = reinterpret_cast<float*>(p.d[which]) + at;
#pragma unroll
    for (int i = 0; i < 32; ++i) w[i] = __float_as_uint(v[i]);
    if (n >= 32 && p.wide) {
#pragma unroll
      for (int i = 0; i < 32; i += 8) st_global_32(d + i, w, i);
    } else {
#pragma unroll
      for (int i = 0; i < 32; i += 4) {
        if (i + 4 <= n) *reinterpret_cast<uint4*>(d + i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
        else {
#pragma unroll
          for (int e = i; e < i + 4; ++e)
            if (e < n) d[e] = v[e];
        }
      }
    }
  } else {
    uint16_t* d = reinterpret_cast<uint16_t*>(p.d[which]) + at;
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = pack_out(bf16, v[2 * i], v[2 * i + 1]);
    if (n >= 32 && p.wide) {
#pragma unroll
      for (int i = 0; i < 16; i += 8) st_global_32(d + 2 * i, w, i);
    } else {
#pragma unroll
      for (int i = 0; i < 32; i += 8) {
        if (i + 8 <= n) *reinterpret_cast<uint4*>(d + i) = make_uint4(w[i / 2], w[i / 2 + 1], w[i / 2 + 2], w[i / 2 + 3]);
        else {
#pragma unroll
          for (int e = i; e < i + 8; ++e)
            if (e < n) d[e] = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
        }
      }
    }
  }
}

// Through shared memory of each epilogue warp, 32 rows x 128 bytes (64 columns): 8 threads per row, so that an instruction writes
// whole lines and not a sector of 32 of them.  0.7 us per 64 columns of a tile instead of 0.9, at the price of a stage of the ring:
// taken for gradients of the weights from up to 512 tokens, which are little but writes (5632 x 2048 from 64 tokens: 16.7 us against
// 18.1; 2048 x 4096 from 300: 17.8 / 18.7; 2731 x 1027 from 777: 19.5 / 19.1); elsewhere the stage is worth more (8-bit products of
// 1500 x 4096 x 1024: 13.7 against 12.2).  The pieces of a row are exchanged by the row's index, against bank conflicts.
__device__ __forceinline__ uint32_t staged_at(uint32_t tile, int r, int piece) { return tile + r * 128 + ((piece ^ (r & 7)) << 4); }
__device__ __forceinline__ void stage_columns(uint32_t tile, int r, int piece0, bool bf16, const float (&v)[32]) {
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const uint32_t w0 = pack_out(bf16, v[g * 8], v[g * 8 + 1]), w1 = pack_out(bf16, v[g * 8 + 2], v[g * 8 + 3]);
    const uint32_t w2 = pack_out(bf16, v[g * 8 + 4], v[g * 8 + 5]), w3 = pack_out(bf16, v[g * 8 + 6], v[g * 8 + 7]);
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(staged_at(tile, r, piece0 + g)), "r"(w0), "r"(w1), "r"(w2), "r"(w3)
                 : "memory");
  }
}
// The staged rows (first: `row`) to result `which` from column `col` on, as far as rows and columns exist.  The whole warp calls.
__device__ __forceinline__ void store_staged(const ProductParams& p, int which, uint32_t tile, int row, int rows, int col, int cols) {
  __syncwarp();
  const int lane = threadIdx.x & 31, piece = lane & 7;
  const int n = cols - (col + piece * 8);                 // columns of this thread's piece that exist, if fewer than 8
  uint16_t* d = reinterpret_cast<uint16_t*>(p.d[which]) + (row + (lane >> 3)) * p.d_stride[which] + col + piece * 8;
  const int64_t step = 4 * p.d_stride[which];
#pragma unroll
  for (int i = 0; i < 8; ++i, d += step) {
    const int r = i * 4 + (lane >> 3);
    if (row + r >= rows || n <= 0) continue;
    uint32_t w[4];
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "r"(staged_at(tile, r, piece)) : "memory");
    if (n >= 8) {
      *reinterpret_cast<uint4*>(d) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int e = 0; e < 7; ++e)
        if (e < n) d[e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
    }
  }
  __syncwarp();                                           // the staging may be written again
}

// int32 sums (as bit patterns) to scaled fp32; lane i holds the scale of column i
template <bool REST>
__device__ __forceinline__ void scale_columns(float (&v)[32], const RowScale& row_scale, float col_scale) {
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    v[i] = __int2float_rn(__float_as_int(v[i])) * row_scale.by * __shfl_sync(0xffffffffu, col_scale, i);
    if constexpr (REST) v[i] *= row_scale.rest;
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
__device__ __forceinline__ int divide(int n, const Divisor& d) { return (int)((__umulhi((uint32_t)n, d.m) + (uint32_t)n) >> d.shift); }
// The `local`-th tile of a pair; false: it has no more (see PairPlan for the order).  Within a list the order is that of tile_coords
// (gemm_tiles.cuh), with the divisions prepared on the host: 4 of them took a third of a microsecond per tile.
__device__ __forceinline__ bool pair_tile(PairTile& t, const PairPlan& plan, int pair, int local, bool grad, int kb) {
  const bool has_more = pair < plan.more;
  const int mine = plan.most + (has_more ? 1 : 0);
  int j = 0, tile = pair + local * plan.pairs;
  if (local >= mine) {
    if (plan.jobs < 2) return false;
    const int i = local - mine;
    j = 1;
    tile = has_more ? i * plan.more + pair : plan.more * plan.share + i * (plan.pairs - plan.more) + (pair - plan.more);
    if (has_more ? i >= plan.share : tile >= plan.job[1].tiles_r * plan.job[1].tiles_c * plan.job[1].batches) return false;
  }
  const PairJob& job = plan.job[j];
  t.kind = job.kind; t.bn = job.bn; t.rows = job.rows; t.cols = job.cols;
  t.batch = divide(tile, job.per_batch);
  int at = tile - t.batch * job.tiles_r * job.tiles_c;
  const int band = divide(at, job.per_band), first_r = band * kGemmBand;
  at -= band * kGemmBand * job.tiles_c;
  if (job.tiles_r - first_r >= kGemmBand) {
    t.tc = at / kGemmBand;
    t.tr = first_r + at % kGemmBand;
  } else {
    t.tc = divide(at, job.tail_rows);
    t.tr = first_r + at - t.tc * (job.tiles_r - first_r);
  }
  if (band & 1) t.tc = job.tiles_c - 1 - t.tc;
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
  const uint32_t ring_bytes = C::XB + plan.y_bytes;           // a k-block: X, then Y
  const uint32_t sStage = sX + plan.stages * ring_bytes;     // [epilogue warps], where results are staged
  const uint32_t sBar = sStage + (GRAD && plan.staged ? 4 * C::GROUPS * C::STAGEB : 0);
  const uint32_t bar_full = sBar;                            // [stages] leader: both CTAs' loads of a stage landed
  const uint32_t bar_empty = sBar + 8 * C::MAXSTAGE;         // [stages] each CTA: its stage was consumed
  const uint32_t bar_acc_full = bar_empty + 8 * C::MAXSTAGE; // [2] each CTA: accumulator complete
  const uint32_t bar_acc_empty = bar_acc_full + 16;          // [2] leader: all epilogue warps of both have read it
  uint8_t* gBar = smem_gen + (sBar - smem_base);
  const uint32_t off_misc = 8 * (2 * C::MAXSTAGE + 4);
  volatile uint32_t* s_tmem_base = reinterpret_cast<volatile uint32_t*>(gBar + off_misc);
  volatile uint32_t* s_abort = reinterpret_cast<volatile uint32_t*>(gBar + off_misc + 4);
  const AbortCtx actx{s_abort, p.status};

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_ctarank();                   // 0 = leader
  const int pair_id = (int)(blockIdx.x >> 1);
  constexpr int KB = I8 ? 128 : 64;                          // elements of the reduction per k-block

  cluster_arrive_started();
  if (tid == 0) {
    for (int i = 0; i < plan.stages; ++i) { mbar_init(bar_full + 8 * i, 2); mbar_init(bar_empty + 8 * i, 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(bar_acc_full + 8 * i, 1); mbar_init(bar_acc_empty + 8 * i, 2 * 4 * C::GROUPS); }
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
      int s = 0, local = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (PairTile t; ok && pair_tile(t, plan, pair_id, local, GRAD, KB); ++local) {
        const int xr = t.tr * C::TM + (int)rank * C::BM;                                    // first of this CTA's rows of X
        const int yr = GATED ? t.tc * t.bn : t.tc * 2 * t.bn + (int)rank * t.bn;            // and of Y
        const uint32_t bytes = C::XB + (GRAD ? (t.bn > 64 ? 2 : 1) * C::SPANB : t.bn * 128);
        for (int i = 0; i < t.nkb; ++i) {
          // every other tile walks the reduction backwards, from the k-blocks that are still in L2 (gemm_sm100.cu)
          const int kb = (local & 1) ? t.nkb - 1 - i : i;
          const int part = GRAD && kb >= t.nkb_part ? 1 : 0;
          const int k = (kb - part * t.nkb_part) * KB;
          if (!mbar_wait(bar_empty + 8 * s, ph ^ 1u, actx, kErrPairEmpty)) { ok = false; break; }
          const uint32_t full = map_to_cta(bar_full + 8 * s, 0);
          const uint32_t x = sX + s * ring_bytes, y = x + C::XB;
          mbar_arrive_expect_tx_cluster(full, bytes);
          if constexpr (GRAD) {      // boxes of 64 x 64
            const CUtensorMap* mx = &maps.x[t.kind == 0 ? part : t.batch];
            const CUtensorMap* my = &maps.y[t.kind == 0 ? part : 2];
            tma_load_3d_pair(x, mx, full, t.kind == 0 ? k : xr, t.kind == 0 ? xr : k, 0);
            tma_load_3d_pair(x + C::SPANB, mx, full, t.kind == 0 ? k : xr + 64, t.kind == 0 ? xr + 64 : k, 0);
            tma_load_3d_pair(y, my, full, yr, k, 0);
            if (t.bn > 64) tma_load_3d_pair(y + C::SPANB, my, full, yr + 64, k, 0);
          } else {
            tma_load_3d_pair(x, &maps.x[0], full, k, xr, 0);
            tma_load_3d_pair(y, &maps.y[GATED ? (int)rank : 0], full, k, yr, 0);
          }
          if (++s == plan.stages) { s = 0; ph ^= 1u; }
        }
      }
    }
  } else if (warp == 1) {
    // UMMA issue: all 32 lanes of the leader's warp run the loop, one elected lane executes the instructions
    if (rank == 0) {
      const uint32_t leader = elect_one();
      const uint32_t fmt = p.bf16 ? kFmtBF16 : kFmtF16;
      int s = 0, local = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (PairTile t; ok && pair_tile(t, plan, pair_id, local, GRAD, KB); ++local) {
        const bool x_mn = GRAD && t.kind == 1;
        const uint32_t idesc = I8 ? make_idesc(2, kFmtS8, kFmtS8, 0, 0, C::TM, 2 * t.bn)
                                  : make_idesc(1, fmt, fmt, x_mn ? 1 : 0, GRAD ? 1 : 0, C::TM, 2 * t.bn);
        // 32 bytes along the reduction, or 16 rows of 128 bytes, per instruction
        const uint32_t xstep = x_mn ? 2048 : 32, xlbo = x_mn ? C::SPANB : 16;
        constexpr uint32_t YSTEP = GRAD ? 2048 : 32, YLBO = GRAD ? C::SPANB : 16;
        const int buf = local & 1;
        if (!mbar_wait_warp(bar_acc_empty + 8 * buf, ((local >> 1) & 1) ^ 1u, actx, kErrPairAccEmpty)) { ok = false; break; }
        tc_fence_after_sync();
        const uint32_t d = tmem_base + buf * C::TN;
        for (int i = 0; i < t.nkb; ++i) {
          if (!mbar_wait_warp(bar_full + 8 * s, ph, actx, kErrPairFull)) { ok = false; break; }
          tc_fence_after_sync();
          const uint64_t a0 = make_smem_desc(sX + s * ring_bytes, xlbo, 1024, kSwizzle128B);
          const uint64_t b0 = make_smem_desc(sX + s * ring_bytes + C::XB, YLBO, 1024, kSwizzle128B);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            const uint64_t a = desc_advance(a0, kk * xstep), bd = desc_advance(b0, kk * YSTEP);
            if constexpr (I8) umma_ss_i8<true>(d, a, bd, idesc, (i | kk) != 0 ? 1u : 0u, leader);
            else umma_ss_e<false, true>(d, a, bd, idesc, (i | kk) != 0 ? 1u : 0u, leader);
          }
          umma_commit_pair_e(bar_empty + 8 * s, (uint16_t)3, leader);      // the stage is free in both CTAs
          if (++s == plan.stages) { s = 0; ph ^= 1u; }
        }
        if (ok) umma_commit_pair_e(bar_acc_full + 8 * buf, (uint16_t)3, leader);
      }
    }
  } else {
    // epilogue warps 2..9 in two groups of four, which take 32 columns of the tile in turn (64 where they are staged); warp w may
    // touch TMEM lanes 32*(w%4) .. +31, a row per thread.
    const int grp = (warp - 2) >> 2;
    const int q = warp & 3;
    const uint32_t lane_base = (uint32_t)(q * 32) << 16;
    const uint32_t leader_acc_empty = map_to_cta(bar_acc_empty, 0);
    const uint32_t stage = sStage + (warp - 2) * C::STAGEB;
    const bool staged = GRAD && plan.staged;
    const int step = staged ? 64 : 32;
    // One tile; false: its accumulator did not come.  `ahead` runs once it has.
    auto finish_tile = [&](const PairTile& t, int local, float row_scale, auto ahead) {
      const int buf = local & 1;
      const int row0 = t.tr * C::TM + (int)rank * C::BM + q * 32, row = row0 + lane;
      const int tcols = GATED ? t.bn : 2 * t.bn, col0 = t.tc * tcols;
      const int end = t.cols - col0 < tcols ? t.cols - col0 : tcols;     // columns of the tile that exist
      const uint32_t acc = tmem_base + lane_base + buf * C::TN;
      const bool inside = row < t.rows;
      [[maybe_unused]] const RowScale rs = split_row_scale(row_scale);
      if (!mbar_wait_warp(bar_acc_full + 8 * buf, (local >> 1) & 1, actx, kErrPairAccFull, 0, p.acc_limit)) return false;
      tc_fence_after_sync();
      ahead();
      // REST: a row of the warp has a scale with a rest.  Tested per tile and not per 32 columns, where the branch alone took 8 % of a
      // gated call of 2048 x 8192 x 256.
      auto columns = [&](auto rest) {
        [[maybe_unused]] constexpr bool REST = decltype(rest)::value;
#pragma unroll 1
        for (int cb = grp * step; cb < end; cb += C::GROUPS * step) {
          const int col = col0 + cb;
          [[maybe_unused]] const int mine = col + lane;          // this lane's column: its scales reach the others by shuffle
          float v[32];
          if constexpr (GATED) {
            float u[32];
            tmem_ld_x32(acc + cb, reinterpret_cast<uint32_t*>(v));
            tmem_ld_x32(acc + t.bn + cb, reinterpret_cast<uint32_t*>(u));
            if constexpr (I8) {
              const float gs = mine < t.cols ? p.col_scale[mine] : 0.f, us = mine < t.cols ? p.col_scale2[mine] : 0.f;
              tmem_wait_ld();
              scale_columns<REST>(v, rs, gs);
              scale_columns<REST>(u, rs, us);
            } else {
              tmem_wait_ld();
            }
            if (p.keep && inside) {
              store_columns(p, 1, row, col, t.cols, v);
              store_columns(p, 2, row, col, t.cols, u);
            }
            gate_columns(p.act, v, u);
            if (inside) store_columns(p, 0, row, col, t.cols, v);
          } else if constexpr (I8) {
            tmem_ld_x32(acc + cb, reinterpret_cast<uint32_t*>(v));
            const float cs = mine < t.cols ? p.col_scale[mine] : 0.f;
            const float bs = p.bias != nullptr && mine < t.cols ? p.bias[mine] : 0.f;
            tmem_wait_ld();
            scale_columns<REST>(v, rs, cs);
            if (p.bias != nullptr) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] += __shfl_sync(0xffffffffu, bs, i);
            }
            if (inside) store_columns(p, 0, row, col, t.cols, v);
          } else {
            const int which = t.kind == 0 ? 0 : 1 + t.batch;
#pragma unroll 1
            for (int h = 0; h < step && cb + h < end; h += 32) {
              tmem_ld_x32(acc + cb + h, reinterpret_cast<uint32_t*>(v));
              tmem_wait_ld();
              if (staged) stage_columns(stage, lane, h / 8, p.bf16, v);
              else if (inside) store_columns(p, which, row, col, t.cols, v);
            }
            if (staged) store_staged(p, which, stage, row0, t.rows, col, end - cb < 64 ? col0 + end : col + 64);
          }
          __syncwarp();
        }
      };
      if constexpr (I8) {
        if (__any_sync(0xffffffffu, rs.rest != 1.f)) columns(std::true_type());
        else columns(std::false_type());
      } else {
        columns(std::false_type());
      }
      // this warp has read the accumulator: the next tile but one may overwrite it
      tc_fence_before_sync();
      mbar_arrive_cluster_warp(leader_acc_empty + 8 * buf);
      return true;
    };
    int local = 0;
    if constexpr (I8) {                // this thread's row scale is read a tile ahead: the first columns wait for it (REST)
      auto row_scale = [&](const PairTile& t) {
        const int row = t.tr * C::TM + (int)rank * C::BM + q * 32 + lane;
        return row < t.rows ? p.row_scale[row] : 0.f;
      };
      PairTile t;
      bool more = pair_tile(t, plan, pair_id, 0, GRAD, KB);
      float scale = more ? row_scale(t) : 0.f;
      for (; more; ++local) {
        const float now = scale;
        PairTile next = t;
        more = pair_tile(next, plan, pair_id, local + 1, GRAD, KB);
        if (!finish_tile(t, local, now, [&] { if (more) scale = row_scale(next); })) break;
        t = next;
      }
    } else {
      bool ok = true;
      for (PairTile t; ok && pair_tile(t, plan, pair_id, local, GRAD, KB); ++local) ok = finish_tile(t, local, 0.f, [] {});
    }
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
int allow_pair_product() { return allow_shared_memory(pair_product_kernel<MODE>, PairCfg::SMEM); }
template <int MODE>
int launch_pair_product(const ProductMaps& maps, const ProductParams& p, PairPlan plan, cudaStream_t stream) {
  using C = PairCfg;
  // narrower tiles leave room for more stages
  int bn = plan.job[0].bn;
  if (plan.jobs > 1 && plan.job[1].bn > bn) bn = plan.job[1].bn;
  plan.y_bytes = MODE == kGrad ? (bn > 64 ? 2 : 1) * C::SPANB : bn * 128;
  const int head = C::HEADB + (MODE == kGrad && plan.staged ? 4 * C::GROUPS * C::STAGEB : 0);
  plan.stages = (C::SMEM - head) / (C::XB + plan.y_bytes);
  if (plan.stages > C::MAXSTAGE) plan.stages = C::MAXSTAGE;
  const size_t smem = head + (size_t)plan.stages * (C::XB + plan.y_bytes);
  return note_cuda(launch_overlapped_in(2, pair_product_kernel<MODE>, dim3((unsigned)(2 * plan.pairs)), dim3(C::NTHREADS), smem,
                                        stream, maps, p, plan), "product launch") == cudaSuccess ? CFK_OK : CFK_ERR_LAUNCH;
}

}  // namespace cfk
