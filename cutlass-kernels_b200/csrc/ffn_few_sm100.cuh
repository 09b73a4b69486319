// The feed-forward products for few tokens (decode, short prompts, short batches), where the weights' traffic or the number of tiles
// counts and not the tensor core's rate.
//
// Operands are exchanged against ffn_pair_sm100.cuh: 128 channels are the M side of the MMA and `tt` tokens (16 to 256) its N
// side, so one token costs a 16-column MMA and not 256 rows.  One CTA per tile of 128 channels x tt tokens; a cluster of `splits` CTAs
// shares the reduction of a tile, because there are as few tiles as cols / 128.  A gated tile reads 128 rows of both weights and
// keeps two accumulators, so that a thread (one channel) has gate and up of an element.  Each weight is read from DRAM once
// while all tokens fit one tile; the tokens are re-read from L2 by every tile.
//
//   warp 0     TMA producer: ring of up to 12 stages of one k-block (128 bytes of the reduction) of weights and tokens
//   warp 1     UMMA issuer, 128 x tt x 32 bytes per instruction
//   warps 2-9  after the last k-block: accumulators -> scales, activation -> the result, channel by lane (64 contiguous
//              bytes of a token's row per warp).  With a split every CTA leaves its accumulators in shared memory
//              ([accumulator][token][channel], the ring is free by then); after a cluster barrier each finishes its share of the
//              tokens, adding the parts in order through distributed shared memory.  Nothing depends on timing.
//
// Bound by DRAM once the first k-blocks have arrived, 2.6 us after the start.  Replayed from a graph: one token through the gated 11264 x
// 4096 in bf16 32 to 33 us (184.6 MB, 5.6 to 5.8 TB/s), 16 tokens in 8 bits 17.5 to 18 us; 48 tokens of 4096 x 11264 in 8 bits 13 us, of which
// 2 to 3 are the exchange of the split.  (As calls of the Python binding 35 to 36, 19.4 and 14 us.)
// A CTA alone on its SM takes a round of 0.19 us per k-block of a product, 0.23 of a gated tile and 0.24 of MN-major weights, with 16 tokens
// or 128: 94 to 168, 148 to 209 and 76 to 141 KB/us.  148 of them get 7.6 TB/s of weights with 16 tokens, and with 128, whose
// re-reads come from L2, 13 TB/s (gated 9.8).  So few tiles split their reduction: one CTA per SM, or a few more, fetch what there is.
//
// Shared memory is sized so that two CTAs fit on an SM where three stages fit in half of it.  Tensor memory never takes a larger
// share of an SM than shared memory does, so residents cannot run out of columns: tcgen05.alloc, which waits without a limit, never
// waits for a CTA that waits for its cluster.
#pragma once
#include "common.cuh"
#include "ffn_act.cuh"
#include "ffn_params.h"
#include "gemm_tiles.cuh"
#include "host_util.h"

namespace cfk {

constexpr int kErrFewFull = 221, kErrFewEmpty = 222, kErrFewAcc = 223;

struct FewCfg {
  static constexpr int MAXSTAGE = kFewMaxStages, NTHREADS = 320, WB = 128 * 128;       // bytes of weights per k-block and accumulator
  static_assert(8 * (2 * MAXSTAGE + 1) + 8 <= 256, "barrier block overflows");
};

template <int ACT>
__device__ __forceinline__ void gate_tokens_by(float (&gate)[8], const float (&up)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) gate[i] = activate<ACT>(gate[i]) * up[i];
}
__device__ __forceinline__ void gate_tokens(int act, float (&gate)[8], const float (&up)[8]) {
  switch (act) {
    case CFK_ACT_SILU: gate_tokens_by<CFK_ACT_SILU>(gate, up); break;
    case CFK_ACT_GELU: gate_tokens_by<CFK_ACT_GELU>(gate, up); break;
    case CFK_ACT_GELU_TANH: gate_tokens_by<CFK_ACT_GELU_TANH>(gate, up); break;
    default: gate_tokens_by<CFK_ACT_RELU>(gate, up); break;
  }
}

// Channel `ch` of 8 tokens from `token` on, `n` of which exist: a warp writes 32 neighbours of each row.
__device__ __forceinline__ void store_tokens(const ProductParams& p, int which, int token, int n, int ch, const float (&v)[8]) {
  const int64_t stride = p.d_stride[which], at = token * stride + ch;
  if (p.out == CFK_FP32) {
    float* d = reinterpret_cast<float*>(p.d[which]) + at;
#pragma unroll
    for (int i = 0; i < 8; ++i, d += stride)
      if (i < n) *d = v[i];
  } else {
    uint16_t* d = reinterpret_cast<uint16_t*>(p.d[which]) + at;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack_out(p.out == CFK_BF16, v[2 * i], v[2 * i + 1]);
#pragma unroll
    for (int i = 0; i < 8; ++i, d += stride)
      if (i < n) *d = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
  }
}

template <int MODE>
__global__ void __launch_bounds__(FewCfg::NTHREADS, 2)
few_product_kernel(const __grid_constant__ ProductMaps maps, const __grid_constant__ ProductParams p,
                   const FewPlan f) {
  using C = FewCfg;
  constexpr bool I8 = MODE == kProductI8 || MODE == kGatedI8;
  constexpr bool GATED = MODE == kGated16 || MODE == kGatedI8;
  constexpr bool W_MN = MODE == kGrad;
  constexpr int NW = GATED ? 2 : 1;                          // weights (and accumulators) of a tile
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t stage_bytes = NW * C::WB + f.tt * 128;      // weights, then tokens
  const uint32_t sRing = smem_base, sBar = smem_base + f.stages * stage_bytes;
  const uint32_t bar_full = sBar, bar_empty = sBar + 8 * C::MAXSTAGE, bar_acc = bar_empty + 8 * C::MAXSTAGE;
  uint8_t* gBar = smem_gen + (sBar - smem_base);
  volatile uint32_t* s_tmem_base = reinterpret_cast<volatile uint32_t*>(gBar + 8 * (2 * C::MAXSTAGE + 1));
  volatile uint32_t* s_abort = s_tmem_base + 1;
  const AbortCtx actx{s_abort, p.status};

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int part = f.splits > 1 ? (int)cluster_ctarank() : 0;
  const int tile = (int)blockIdx.x / f.splits, tile_ch = tile / f.tiles_tok, tile_tok = tile - tile_ch * f.tiles_tok;
  const int ch0 = tile_ch * 128, tok0 = tile_tok * f.tt;
  const int ntok = p.rows - tok0 < f.tt ? p.rows - tok0 : f.tt;
  constexpr int KB = I8 ? 128 : 64;                          // elements of the reduction per k-block
  const int nkb_part = (p.reduce + KB - 1) / KB;
  const int nkb_all = MODE == kGrad ? 2 * nkb_part : nkb_part;
  const int kb0 = (int)((long long)nkb_all * part / f.splits), kb1 = (int)((long long)nkb_all * (part + 1) / f.splits);
  const int acc_cols = (f.tt + 31) & ~31;                    // tensor-memory columns from one accumulator to the next
  uint32_t ncols = 32;
  while (ncols < (uint32_t)(NW * acc_cols)) ncols *= 2;

  if (f.splits > 1) cluster_arrive_started();
  if (tid == 0) {
    for (int i = 0; i < f.stages; ++i) { mbar_init(bar_full + 8 * i, 1); mbar_init(bar_empty + 8 * i, 1); }
    mbar_init(bar_acc, 1);
    *s_abort = 0u;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(const_cast<uint32_t*>(s_tmem_base)), ncols);
    tmem_relinquish();
    grid_dependency_launch();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&maps.x[0]);
    tma_prefetch_desc(&maps.y[0]);
    if (GATED) tma_prefetch_desc(&maps.y[1]);
  }
  grid_dependency_wait();
  tc_fence_before_sync();
  bool skip;
  if (f.splits > 1) {
    __syncwarp();
    cluster_wait_started();
    skip = cluster_should_skip(p.status, f.splits);          // one decision for the cluster
  } else {
    skip = cta_should_skip(p.status);
  }
  tc_fence_after_sync();
  const uint32_t tmem_base = *s_tmem_base;
  if (skip) {
    if (warp == 1) tmem_dealloc(tmem_base, ncols);
    return;
  }

  if (warp == 0) {
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        const int seg = MODE == kGrad && kb >= nkb_part ? 1 : 0;
        const int k = (kb - seg * nkb_part) * KB;
        if (!mbar_wait(bar_empty + 8 * s, ph ^ 1u, actx, kErrFewEmpty)) break;
        const uint32_t full = bar_full + 8 * s, at = sRing + s * stage_bytes;
        mbar_arrive_expect_tx(full, stage_bytes);
        if constexpr (W_MN) {
          tma_load_3d(at, &maps.y[seg], full, ch0, k, 0);
          tma_load_3d(at + C::WB / 2, &maps.y[seg], full, ch0 + 64, k, 0);
        } else {
          tma_load_3d(at, &maps.y[0], full, k, ch0, 0);
          if constexpr (GATED) tma_load_3d(at + C::WB, &maps.y[1], full, k, ch0, 0);
        }
        tma_load_3d(at + NW * C::WB, &maps.x[seg], full, k, tok0, 0);
        if (++s == f.stages) { s = 0; ph ^= 1u; }
      }
    }
  } else if (warp == 1) {
    const uint32_t leader = elect_one();
    const uint32_t fmt = p.bf16 ? kFmtBF16 : kFmtF16;
    const uint32_t idesc = I8 ? make_idesc(2, kFmtS8, kFmtS8, 0, 0, 128, (uint32_t)f.tt)
                              : make_idesc(1, fmt, fmt, W_MN ? 1 : 0, 0, 128, (uint32_t)f.tt);
    constexpr uint32_t WSTEP = W_MN ? 2048 : 32;
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!mbar_wait_warp(bar_full + 8 * s, ph, actx, kErrFewFull)) { ok = false; break; }
      tc_fence_after_sync();
      const uint32_t at = sRing + s * stage_bytes;
      const uint64_t b0 = make_smem_desc(at + NW * C::WB, 16, 1024, kSwizzle128B);
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const uint64_t a0 = make_smem_desc(at + w * C::WB, W_MN ? C::WB / 2 : 16, 1024, kSwizzle128B);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          const uint32_t acc = kb != kb0 || kk != 0 ? 1u : 0u, d = tmem_base + w * acc_cols;
          const uint64_t a = desc_advance(a0, kk * WSTEP), b = desc_advance(b0, kk * 32);
          if constexpr (I8) umma_ss_i8<false>(d, a, b, idesc, acc, leader);
          else umma_ss_e<false, false>(d, a, b, idesc, acc, leader);
        }
      }
      umma_commit_e<false>(bar_empty + 8 * s, leader);
      if (++s == f.stages) { s = 0; ph ^= 1u; }
    }
    if (ok) umma_commit_e<false>(bar_acc, leader);
  }

  const int q = warp & 3, r = q * 32 + lane, ch = ch0 + r;   // epilogue: this thread's TMEM lane and channel
  const int grp = (warp - 2) >> 2;                           // two groups of four warps take turns of 8 tokens
  const bool epilogue = warp >= 2;
  float cs = 0.f, cs2 = 0.f, bias = 0.f;
  bool done = false;
  if (epilogue) {
    if constexpr (I8) {
      if (ch < p.cols) {
        cs = p.col_scale[ch];
        if constexpr (GATED) cs2 = p.col_scale2[ch];
        else if (p.bias != nullptr) bias = p.bias[ch];
      }
    }
    done = mbar_wait_warp(bar_acc, 0, actx, kErrFewAcc, 0, p.acc_limit);
    tc_fence_after_sync();
  }

  // the results of 8 tokens of the tile from t0 on, `n` of which exist, from their complete sums (fp32 or int32)
  auto finish = [&](int t0, int n, const uint32_t (&s0)[8], const uint32_t (&s1)[8]) {
    const int token = tok0 + t0;
    float v[8], u[8];
    if constexpr (I8) {
      const RowScale rs = split_row_scale(lane < n ? p.row_scale[token + lane] : 0.f);     // n <= 8
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float rsi = __shfl_sync(0xffffffffu, rs.by, i);
        v[i] = __int2float_rn((int)s0[i]) * rsi * cs;
        if constexpr (GATED) u[i] = __int2float_rn((int)s1[i]) * rsi * cs2;
      }
      if (__any_sync(0xffffffffu, rs.rest != 1.f)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float rest = __shfl_sync(0xffffffffu, rs.rest, i);
          v[i] *= rest;
          if constexpr (GATED) u[i] *= rest;
        }
      }
      if constexpr (!GATED) {
        if (p.bias != nullptr) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] += bias;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = __uint_as_float(s0[i]);
        if constexpr (GATED) u[i] = __uint_as_float(s1[i]);
      }
    }
    if (ch < p.cols) {
      if constexpr (GATED) {
        if (p.keep) {
          store_tokens(p, 1, token, n, ch, v);
          store_tokens(p, 2, token, n, ch, u);
        }
        gate_tokens(p.act, v, u);
      }
      store_tokens(p, 0, token, n, ch, v);
    }
    __syncwarp();
  };

  const uint32_t lane_base = tmem_base + ((uint32_t)(q * 32) << 16);
  if (f.splits == 1) {
    if (done) {
#pragma unroll 1
      for (int t0 = 8 * grp; t0 < ntok; t0 += 16) {
        uint32_t a[8], b[8];
        tmem_ld_x8(lane_base + t0, a);
        if constexpr (GATED) tmem_ld_x8(lane_base + acc_cols + t0, b);
        tmem_wait_ld();
        finish(t0, ntok - t0 < 8 ? ntok - t0 : 8, a, b);
      }
    }
  } else {
    if (done) {
#pragma unroll 1
      for (int c = 8 * grp; c < NW * acc_cols; c += 16) {
        const int t0 = c < acc_cols ? c : c - acc_cols;
        if (t0 >= ntok) continue;
        uint32_t a[8];
        tmem_ld_x8(lane_base + c, a);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (t0 + i < ntok) asm volatile("st.shared.b32 [%0], %1;" ::"r"(sRing + (c + i) * 512 + r * 4), "r"(a[i]) : "memory");
      }
    }
    __syncwarp();
    cluster_sync_all();            // every CTA's accumulators are in its shared memory
    if (done && !*s_abort) {
      const int t1 = ntok * (part + 1) / f.splits;
#pragma unroll 1
      for (int t0 = ntok * part / f.splits + 8 * grp; t0 < t1; t0 += 16) {
        const int n = t1 - t0 < 8 ? t1 - t0 : 8;
        uint32_t a[8], b[8];
        // a few tokens at a time (as registers allow), the parts of all CTAs in flight together: a read takes about half a microsecond
        constexpr int STEP = GATED ? 2 : 4;
        auto gather = [&](uint32_t (&sum)[8], int first) {
          const uint32_t from = sRing + first * 512 + r * 4;
#pragma unroll
          for (int g = 0; g < 8; g += STEP) {
            if (g >= n) break;
            float v[8][STEP];
#pragma unroll
            for (int o = 0; o < 8; ++o)
              if (o < f.splits) {
#pragma unroll
                for (int i = 0; i < STEP; ++i)
                  if (g + i < n) v[o][i] = ld_shared_cluster_f32(map_to_cta(from, (uint32_t)o) + (g + i) * 512);
              }
#pragma unroll
            for (int i = 0; i < STEP; ++i) sum[g + i] = __float_as_uint(v[0][i]);
#pragma unroll
            for (int o = 1; o < 8; ++o)      // in the order of the reduction
              if (o < f.splits) {
#pragma unroll
                for (int i = 0; i < STEP; ++i)
                  sum[g + i] = I8 ? sum[g + i] + __float_as_uint(v[o][i])
                                  : __float_as_uint(__uint_as_float(sum[g + i]) + v[o][i]);
              }
          }
        };
        gather(a, t0);
        if constexpr (GATED) gather(b, acc_cols + t0);
        finish(t0, n, a, b);
      }
    }
  }

  settle_if_aborted(s_abort);
  tc_fence_before_sync();
  __syncthreads();
  if (f.splits > 1) cluster_sync_all();     // no CTA leaves while another may still read its shared memory
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, ncols);
  }
}

template <int MODE>
int allow_few_product() { return allow_shared_memory(few_product_kernel<MODE>, kFewSmemFull); }
template <int MODE>
int launch_few_product(const ProductMaps& maps, const ProductParams& p, const FewPlan& f, cudaStream_t stream) {
  const dim3 grid((unsigned)(f.tiles_ch * f.tiles_tok * f.splits));
  const size_t smem = kFewHead + (size_t)f.stages * (few_weights(MODE) * FewCfg::WB + f.tt * 128);
  return note_cuda(launch_overlapped_in(f.splits, few_product_kernel<MODE>, grid, dim3(FewCfg::NTHREADS), smem, stream, maps, p, f),
                   "few-token product launch") == cudaSuccess ? CFK_OK : CFK_ERR_LAUNCH;
}

}  // namespace cfk
