// The feed-forward products on CTA pairs: tiles of 256 rows x 256 columns of accumulator, as in gemm_sm100.cu, for operands and
// results that a plain GEMM does not have.
//
//   kProductI8   8-bit integers (kind::i8, 128 elements per 128-byte k-block, int32 sums), scaled per row and column at the end
//   kGated16/I8  the leader's half of the accumulator columns is the gate projection and its peer's half the up projection: each
//                CTA loads 128 rows of ONE of the two weights, so the pair's 256 columns hold gate and up of the same 128 columns
//                of h, and the epilogue has both of an element in one thread.  x is read once for the two products.
//   kGradX       one reduction over the channels of w_gate and then of w_up: dx leaves the tensor core summed.  The weights are
//                stored with the model's width contiguous, which is the column of dx: they are MN-major operands.
//   kGradW       reduction over the tokens, along which neither operand is contiguous: both are MN-major.
//
// Roles, ring, tensor-memory double buffer and store path are those of gemm_kernel: warp 0 TMA, warp 1 of the leader
// UMMA (cta_group::2), warps 2-5 epilogue with two alternating staging tiles and TMA stores that clip at the result's edges.
// An MN-major operand lands as two spans of 64 columns, [span][64 k-rows][128 bytes], each with the 128-byte swizzle; what lies
// behind a matrix is zero-filled in both operands, so ragged reductions need no mask.
//
// Bound by the tensor core: 512 clk of MMA per k-block of 128 bytes against 32 KB of loads per SM and, in the gated modes, an
// epilogue of two special-function operations per element of h that runs beside the next tile's main loop.
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
  static constexpr int STAGEB = 128 * 128;                         // output staging tile: 128 rows x 128 bytes
  static constexpr int SMEM_BYTES = 1024 + NSTAGE * (XB + YB) + 2 * STAGEB + 256;
  static constexpr int NTHREADS = 192;
  static_assert(8 * (2 * NSTAGE + 8) + 8 <= 256, "barrier block overflows");
};

// 32 values of a row as 16-byte pieces `piece0`.. of a 128-byte row of a staging tile: piece index XOR (row & 7), the 128-byte
// swizzle that the TMA store undoes
__device__ __forceinline__ void stage_row16(uint32_t row_addr, int r, int piece0, bool bf16, const float (&v)[32]) {
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const uint32_t w0 = pack_out(bf16, v[g * 8], v[g * 8 + 1]), w1 = pack_out(bf16, v[g * 8 + 2], v[g * 8 + 3]);
    const uint32_t w2 = pack_out(bf16, v[g * 8 + 4], v[g * 8 + 5]), w3 = pack_out(bf16, v[g * 8 + 6], v[g * 8 + 7]);
    const uint32_t piece = (uint32_t)(piece0 + g) ^ (uint32_t)(r & 7);
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row_addr + piece * 16), "r"(w0), "r"(w1), "r"(w2), "r"(w3)
                 : "memory");
  }
}
__device__ __forceinline__ void stage_row32(uint32_t row_addr, int r, const float (&v)[32]) {
#pragma unroll
  for (int g = 0; g < 8; ++g) {
    const uint32_t piece = (uint32_t)g ^ (uint32_t)(r & 7);
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row_addr + piece * 16), "r"(__float_as_uint(v[g * 4])),
                 "r"(__float_as_uint(v[g * 4 + 1])), "r"(__float_as_uint(v[g * 4 + 2])), "r"(__float_as_uint(v[g * 4 + 3]))
                 : "memory");
  }
}

// The columns of a row behind the last whole 16 bytes (see ProductParams::whole), read back from this thread's own row of the
// staging tile, whose first column is `col`.
__device__ __forceinline__ void store_rest(const ProductParams& p, int which, bool out32, uint32_t row_addr, int r, int row, int col) {
  const int esz = out32 ? 4 : 2;
  const int end = p.cols < col + 128 / esz ? p.cols : col + 128 / esz;
  for (int c = p.whole > col ? p.whole : col; c < end; ++c) {
    const uint32_t byte = (uint32_t)((c - col) * esz);
    const uint32_t from = row_addr + (((byte >> 4) ^ (uint32_t)(r & 7)) << 4) + (byte & 15u);
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

template <int MODE>
__global__ void __launch_bounds__(192, 1)
pair_product_kernel(const __grid_constant__ ProductMaps maps, const ProductParams p) {
  using C = PairCfg;
  constexpr bool I8 = MODE == kProductI8 || MODE == kGatedI8;
  constexpr bool GATED = MODE == kGated16 || MODE == kGatedI8;
  constexpr bool X_MN = MODE == kGradW, Y_MN = MODE == kGradX || MODE == kGradW;
  constexpr int TCOLS = GATED ? 128 : 256;            // columns of the result per tile
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t sX = smem_base;
  const uint32_t sY = smem_base + C::NSTAGE * C::XB;
  const uint32_t sStage = sY + C::NSTAGE * C::YB;            // [2] output staging tiles
  const uint32_t sBar = sStage + 2 * C::STAGEB;
  const uint32_t bar_full = sBar;                            // [NSTAGE] leader: both CTAs' loads of a stage landed
  const uint32_t bar_empty = sBar + 8 * C::NSTAGE;           // [NSTAGE] each CTA: its stage was consumed
  const uint32_t bar_acc_full = bar_empty + 8 * C::NSTAGE;   // [2] each CTA: accumulator complete
  const uint32_t bar_acc_empty = bar_acc_full + 16;          // [2] leader: both epilogues have read it
  const uint32_t bar_staged = bar_acc_empty + 16;            // [2] a staging tile is complete (4 epilogue warps)
  const uint32_t bar_stage_free = bar_staged + 16;           // [2] the TMA store has read a staging tile
  uint8_t* gBar = smem_gen + (sBar - smem_base);
  const uint32_t off_misc = 8 * (2 * C::NSTAGE + 8);
  volatile uint32_t* s_tmem_base = reinterpret_cast<volatile uint32_t*>(gBar + off_misc);
  volatile uint32_t* s_abort = reinterpret_cast<volatile uint32_t*>(gBar + off_misc + 4);
  const AbortCtx actx{s_abort, p.status};

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_ctarank();                   // 0 = leader
  const int pair_id = (int)(blockIdx.x >> 1), n_pairs = (int)(gridDim.x >> 1);
  const int total_tiles = p.tiles_r * p.tiles_c * p.batches;
  constexpr int KB = I8 ? 128 : 64;                          // elements of the reduction per k-block
  const int nkb_part = (p.reduce + KB - 1) / KB;
  const int nkb = MODE == kGradX ? 2 * nkb_part : nkb_part;

  cluster_arrive_started();
  if (tid == 0) {
    for (int i = 0; i < C::NSTAGE; ++i) { mbar_init(bar_full + 8 * i, 2); mbar_init(bar_empty + 8 * i, 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(bar_acc_full + 8 * i, 1); mbar_init(bar_acc_empty + 8 * i, 256); }
    for (int i = 0; i < 2; ++i) { mbar_init(bar_staged + 8 * i, 4); mbar_init(bar_stage_free + 8 * i, 1); }
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
      for (int tile = pair_id; tile < total_tiles && ok; tile += n_pairs, ++local) {
        int tr, tc, b;
        tile_coords(tile, p.tiles_r, p.tiles_c, tr, tc, b);
        const int xr = tr * C::TM + (int)rank * C::BM;                             // first of this CTA's rows of X
        const int yr = GATED ? tc * TCOLS : tc * TCOLS + (int)rank * C::BN;        // and of Y
        for (int i = 0; i < nkb; ++i, ++idx) {
          // every other tile walks the reduction backwards, from the k-blocks that are still in L2 (gemm_sm100.cu)
          const int kb = (local & 1) ? nkb - 1 - i : i;
          const int part = MODE == kGradX && kb >= nkb_part ? 1 : 0;
          const int k = (kb - part * nkb_part) * KB;
          const int s = idx % C::NSTAGE;
          const uint32_t ph = (idx / C::NSTAGE) & 1;
          if (!mbar_wait(bar_empty + 8 * s, ph ^ 1u, actx, kErrPairEmpty)) { ok = false; break; }
          const uint32_t full = map_to_cta(bar_full + 8 * s, 0);
          mbar_arrive_expect_tx_cluster(full, C::XB + C::YB);
          const CUtensorMap* mx = &maps.x[MODE == kGradX ? part : (MODE == kGradW ? b : 0)];
          const CUtensorMap* my = &maps.y[MODE == kGradX ? part : (GATED ? (int)rank : 0)];
          if constexpr (X_MN) {
            tma_load_3d_pair(sX + s * C::XB, mx, full, xr, k, 0);
            tma_load_3d_pair(sX + s * C::XB + C::XB / 2, mx, full, xr + 64, k, 0);
          } else {
            tma_load_3d_pair(sX + s * C::XB, mx, full, k, xr, 0);
          }
          if constexpr (Y_MN) {
            tma_load_3d_pair(sY + s * C::YB, my, full, yr, k, 0);
            tma_load_3d_pair(sY + s * C::YB + C::YB / 2, my, full, yr + 64, k, 0);
          } else {
            tma_load_3d_pair(sY + s * C::YB, my, full, k, yr, 0);
          }
        }
      }
    }
  } else if (warp == 1) {
    // UMMA issue: all 32 lanes of the leader's warp run the loop, one elected lane executes the instructions
    if (rank == 0) {
      const uint32_t leader = elect_one();
      const uint32_t fmt = p.bf16 ? kFmtBF16 : kFmtF16;
      const uint32_t idesc = I8 ? make_idesc(2, kFmtS8, kFmtS8, 0, 0, C::TM, C::TN)
                                : make_idesc(1, fmt, fmt, X_MN ? 1 : 0, Y_MN ? 1 : 0, C::TM, C::TN);
      // 32 bytes along the reduction, or 16 rows of 128 bytes, per instruction
      constexpr uint32_t XSTEP = X_MN ? 2048 : 32, YSTEP = Y_MN ? 2048 : 32;
      int idx = 0, local = 0;
      bool ok = true;
      for (int tile = pair_id; tile < total_tiles && ok; tile += n_pairs, ++local) {
        const int buf = local & 1;
        if (!mbar_wait_warp(bar_acc_empty + 8 * buf, ((local >> 1) & 1) ^ 1u, actx, kErrPairAccEmpty)) { ok = false; break; }
        tc_fence_after_sync();
        const uint32_t d = tmem_base + buf * C::TN;
        for (int i = 0; i < nkb; ++i, ++idx) {
          const int s = idx % C::NSTAGE;
          if (!mbar_wait_warp(bar_full + 8 * s, (idx / C::NSTAGE) & 1, actx, kErrPairFull)) { ok = false; break; }
          tc_fence_after_sync();
          const uint64_t a0 = make_smem_desc(sX + s * C::XB, X_MN ? C::XB / 2 : 16, 1024, kSwizzle128B);
          const uint64_t b0 = make_smem_desc(sY + s * C::YB, Y_MN ? C::YB / 2 : 16, 1024, kSwizzle128B);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            const uint64_t a = desc_advance(a0, kk * XSTEP), bd = desc_advance(b0, kk * YSTEP);
            if constexpr (I8) umma_ss_i8<true>(d, a, bd, idesc, (i | kk) != 0 ? 1u : 0u, leader);
            else umma_ss_e<false, true>(d, a, bd, idesc, (i | kk) != 0 ? 1u : 0u, leader);
          }
          umma_commit_pair_e(bar_empty + 8 * s, (uint16_t)3, leader);      // the stage is free in both CTAs
        }
        if (ok) umma_commit_pair_e(bar_acc_full + 8 * buf, (uint16_t)3, leader);
      }
    }
  } else {
    // epilogue warps 2..5; warp w may touch TMEM lanes 32*(w%4) .. +31.  A tile leaves in chunks of 128 bytes per row, each
    // through one of two staging tiles; with `keep` the chunks of h, gate and up follow each other.
    const int q = warp & 3;
    const int r = q * 32 + lane;                       // row within this CTA's 128 rows
    const uint32_t lane_base = (uint32_t)(q * 32) << 16;
    const uint32_t leader_acc_empty = map_to_cta(bar_acc_empty, 0);
    const bool out32 = MODE == kProductI8 && p.out == CFK_FP32, out_bf16 = p.out == CFK_BF16;
    const int ccols = out32 ? 32 : 64;                 // columns per chunk
    const int kinds = GATED && p.keep ? 3 : 1;         // chunks per 64 columns: h, gate, up
    const int nchunk = TCOLS / ccols * kinds;
    const bool storer = (warp == 2 && lane == 0);
    int local = 0;
    uint32_t n = 0;                                    // chunks staged so far: chunk n uses staging tile n & 1
    bool ok = true;
    for (int tile = pair_id; tile < total_tiles && ok; tile += n_pairs, ++local) {
      int tr, tc, b;
      tile_coords(tile, p.tiles_r, p.tiles_c, tr, tc, b);
      const int buf = local & 1;
      const int row = tr * C::TM + (int)rank * C::BM + r;
      const int col0 = tc * TCOLS;
      const uint32_t acc = tmem_base + lane_base + buf * C::TN;
      float rs = 0.f;
      if constexpr (I8) rs = row < p.rows ? __ldg(p.row_scale + row) : 0.f;
      ok = mbar_wait_warp(bar_acc_full + 8 * buf, (local >> 1) & 1, actx, kErrPairAccFull);
      if (!ok) break;
      tc_fence_after_sync();
#pragma unroll 1
      for (int ch = 0; ch < nchunk; ++ch, ++n) {
        const int kind = kinds == 1 ? 0 : ch % 3;
        const int cc = (kinds == 1 ? ch : ch / 3) * ccols;     // first column of the chunk within the tile
        const uint32_t sb = n & 1u;
        const uint32_t stage = sStage + sb * C::STAGEB;
        if (n >= 2u) {   // the store that last used this staging tile has read it
          ok = mbar_wait_warp(bar_stage_free + 8 * sb, ((n >> 1) & 1u) ^ 1u, actx, kErrPairStageFree);
          if (!ok) break;
        }
        const uint32_t row_addr = stage + r * 128;
#pragma unroll 1
        for (int hh = 0; hh < ccols / 32; ++hh) {              // 32 accumulator columns at a time
          const int cb = cc + hh * 32;
          const int col = col0 + cb + lane;                    // this lane's column: its scales reach the others by shuffle
          float v[32];
          if constexpr (GATED) {
            float gs = 1.f, us = 1.f;
            if constexpr (I8) {
              gs = col < p.cols ? __ldg(p.col_scale + col) : 0.f;
              us = col < p.cols ? __ldg(p.col_scale2 + col) : 0.f;
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
              tmem_ld_x32(acc + 128 + cb, w);
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
            stage_row16(row_addr, r, hh * 4, out_bf16, v);
          } else {
            uint32_t w[32];
            tmem_ld_x32(acc + cb, w);
            tmem_wait_ld();
            if constexpr (I8) {
              const float cs = col < p.cols ? __ldg(p.col_scale + col) : 0.f;
              const float bs = p.bias != nullptr && col < p.cols ? __ldg(p.bias + col) : 0.f;
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = __int2float_rn((int)w[i]) * rs * __shfl_sync(0xffffffffu, cs, i);
              if (p.bias != nullptr) {
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] += __shfl_sync(0xffffffffu, bs, i);
              }
              if (out32) stage_row32(row_addr, r, v);
              else stage_row16(row_addr, r, hh * 4, out_bf16, v);
            } else {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(w[i]);
              stage_row16(row_addr, r, hh * 4, out_bf16, v);
            }
          }
        }
        if (row < p.rows && col0 + cc + ccols > p.whole) store_rest(p, MODE == kGradW ? b : kind, out32, row_addr, r, row, col0 + cc);
        if (ch == nchunk - 1) {   // the accumulator has been read: the next tile but one may overwrite it
          tc_fence_before_sync();
          mbar_arrive_cluster(leader_acc_empty + 8 * buf);
        }
        fence_proxy_async_smem();
        mbar_arrive_warp(bar_staged + 8 * sb);
        if (storer) {
          if (!mbar_wait(bar_staged + 8 * sb, (n >> 1) & 1u, actx, kErrPairStaged)) { ok = false; }
          else {
            if (p.whole > 0) tma_store_3d(&maps.d[MODE == kGradW ? b : kind], stage, col0 + cc, tr * C::TM + (int)rank * C::BM, 0);
            tma_store_commit();
            tma_store_wait_read1();            // every store but this one has read its staging tile
            if (n >= 1u) mbar_arrive(bar_stage_free + 8 * (sb ^ 1u));
          }
        }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
      }
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
int launch_pair_product(const ProductMaps& maps, const ProductParams& p, cudaStream_t stream) {
  using C = PairCfg;
  static thread_local int attr_dev = -1;
  static thread_local int sm_count = 0;
  int dev = 0;
  if (note_cuda(cudaGetDevice(&dev), "cudaGetDevice") != cudaSuccess) return CFK_ERR_NO_DRIVER;
  if (attr_dev != dev) {
    if (note_cuda(cudaFuncSetAttribute(pair_product_kernel<MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES),
                  "cudaFuncSetAttribute(product smem)") != cudaSuccess)
      return CFK_ERR_LAUNCH;
    if (note_cuda(cudaDeviceGetAttribute(&sm_count, cudaDevAttrMultiProcessorCount, dev), "sm count") != cudaSuccess)
      return CFK_ERR_LAUNCH;
    attr_dev = dev;
  }
  const long long total = (long long)p.tiles_r * p.tiles_c * p.batches;
  const long long pairs = total < sm_count / 2 ? total : sm_count / 2;
  return note_cuda(launch_overlapped_in(2, pair_product_kernel<MODE>, dim3((unsigned)(2 * pairs)), dim3(C::NTHREADS), C::SMEM_BYTES,
                                        stream, maps, p), "product launch") == cudaSuccess ? CFK_OK : CFK_ERR_LAUNCH;
}

}  // namespace cfk
