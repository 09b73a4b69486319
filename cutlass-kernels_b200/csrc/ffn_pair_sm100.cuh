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
// two groups of four epilogue warps, which write whole sectors from registers.  (A TMA store writes whole 16-byte pieces, so behind
// the last element of a row it would put zeros up to the next multiple of 16 bytes; and the hand-over of its staging tiles took 0.6 us
// per 32 columns, most of a tile whose reduction is short.)
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

constexpr int kErrPairFull = 211, kErrPairEmpty = 212, kErrPairAccFull = 213, kErrPairAccEmpty = 214;

struct PairCfg {
  static constexpr int TM = 256, TN = 256, BM = 128, BN = 128;     // tile of the pair; rows of X and of Y per CTA
  static constexpr int XB = BM * 128, YB = BN * 128;               // bytes per k-block
  static constexpr int NSTAGE = 7;
  static constexpr int GROUPS = 2;                                 // of four epilogue warps
  static constexpr int SMEM_BYTES = 1024 + NSTAGE * (XB + YB) + 256;
  static constexpr int NTHREADS = 64 + GROUPS * 128;
  static_assert(8 * (2 * NSTAGE + 4) + 8 <= 256, "barrier block overflows");
};

// 32 columns of a row, from `col` on, as far as they exist.  A thread writes whole 32-byte sectors where rows start at multiples of
// 32 bytes (`wide`), and nothing behind the row's end.
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
  const uint32_t sBar = sY + C::NSTAGE * C::YB;
  const uint32_t bar_full = sBar;                            // [NSTAGE] leader: both CTAs' loads of a stage landed
  const uint32_t bar_empty = sBar + 8 * C::NSTAGE;           // [NSTAGE] each CTA: its stage was consumed
  const uint32_t bar_acc_full = bar_empty + 8 * C::NSTAGE;   // [2] each CTA: accumulator complete
  const uint32_t bar_acc_empty = bar_acc_full + 16;          // [2] leader: all epilogue warps of both have read it
  uint8_t* gBar = smem_gen + (sBar - smem_base);
  const uint32_t off_misc = 8 * (2 * C::NSTAGE + 4);
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
    // epilogue warps 2..9 in two groups of four, which take 32 columns of the tile in turn; warp w may touch TMEM lanes
    // 32*(w%4) .. +31, a row per thread.
    const int grp = (warp - 2) >> 2;
    const int q = warp & 3;
    const int r = q * 32 + lane;                       // row within this CTA's 128 rows
    const uint32_t lane_base = (uint32_t)(q * 32) << 16;
    const uint32_t leader_acc_empty = map_to_cta(bar_acc_empty, 0);
    int local = 0;
    bool ok = true;
    for (PairTile t; ok && pair_tile(t, plan, pair_id, local, GRAD, KB); ++local) {
      const int buf = local & 1;
      const int row = t.tr * C::TM + (int)rank * C::BM + r;
      const int tcols = GATED ? t.bn : 2 * t.bn, col0 = t.tc * tcols;
      const int end = t.cols - col0 < tcols ? t.cols - col0 : tcols;     // columns of the tile that exist
      const uint32_t acc = tmem_base + lane_base + buf * C::TN;
      const bool inside = row < t.rows;
      float rs = 0.f;
      if constexpr (I8) rs = inside ? p.row_scale[row] : 0.f;
      ok = mbar_wait_warp(bar_acc_full + 8 * buf, (local >> 1) & 1, actx, kErrPairAccFull);
      if (!ok) break;
      tc_fence_after_sync();
#pragma unroll 1
      for (int cb = grp * 32; cb < end; cb += C::GROUPS * 32) {
        const int col = col0 + cb, mine = col + lane;          // this lane's column: its scales reach the others by shuffle
        float v[32];
        if constexpr (GATED) {
          float u[32];
          uint32_t w[32], x[32];
          tmem_ld_x32(acc + cb, w);
          tmem_ld_x32(acc + t.bn + cb, x);
          if constexpr (I8) {
            const float gs = mine < t.cols ? p.col_scale[mine] : 0.f;
            const float us = mine < t.cols ? p.col_scale2[mine] : 0.f;
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              v[i] = __int2float_rn((int)w[i]) * rs * __shfl_sync(0xffffffffu, gs, i);
              u[i] = __int2float_rn((int)x[i]) * rs * __shfl_sync(0xffffffffu, us, i);
            }
          } else {
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) { v[i] = __uint_as_float(w[i]); u[i] = __uint_as_float(x[i]); }
          }
          if (p.keep && inside) {
            store_columns(p, 1, row, col, t.cols, v);
            store_columns(p, 2, row, col, t.cols, u);
          }
          gate_columns(p.act, v, u);
          if (inside) store_columns(p, 0, row, col, t.cols, v);
        } else {
          uint32_t w[32];
          tmem_ld_x32(acc + cb, w);
          if constexpr (I8) {
            const float cs = mine < t.cols ? p.col_scale[mine] : 0.f;
            const float bs = p.bias != nullptr && mine < t.cols ? p.bias[mine] : 0.f;
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __int2float_rn((int)w[i]) * rs * __shfl_sync(0xffffffffu, cs, i);
            if (p.bias != nullptr) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] += __shfl_sync(0xffffffffu, bs, i);
            }
          } else {
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(w[i]);
          }
          if (inside) store_columns(p, GRAD ? (t.kind == 0 ? 0 : 1 + t.batch) : 0, row, col, t.cols, v);
        }
        __syncwarp();
      }
      // this warp has read the accumulator: the next tile but one may overwrite it
      tc_fence_before_sync();
      mbar_arrive_cluster_warp(leader_acc_empty + 8 * buf);
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
