// Entry points of the feed-forward operators (include/cfk_b200.h): argument checks, descriptors and choice of kernel, and the
// elementwise part of the gated block's backward pass.
#include <cmath>
#include <cstring>
#include <utility>

#include "common.cuh"
#include "element_io.cuh"
#include "ffn_act.cuh"
#include "ffn_params.h"
#include "gemm_tiles.cuh"
#include "host_util.h"

namespace cfk {

static int64_t packed(int64_t stride, int cols) { return stride == 0 ? cols : stride; }

// dgate = dh * up * act'(gate), dup = dh * act(gate).  Memory bound: three 16-bit values in, two out, 16 bytes per access, a thread
// reads its elements of all three before it writes, so the results may take the place of gate and up.  8192 x 11264 bf16, replayed from
// a graph: SiLU 134 us, 6.9 TB/s, in place 140, with six blocks per SM (five: 146); GELU 228, its erfc.
// IN_PLACE: behind a wait that gave up nothing is written, as by the products that follow, since it would overwrite the inputs of the
// call when it is repeated.  The word is read beside the elements, so the test costs a barrier and not a memory latency: 0.5 us of 777 x
// 2731.  (Every thread reading it: 146 us for the 140 above.)
template <int DT, int ACT, bool IN_PLACE>
__global__ void __launch_bounds__(256, 6)
gate_grad_kernel(const uint16_t* dh, const uint16_t* gate, const uint16_t* up, uint16_t* dgate, uint16_t* dup, int64_t dh_stride,
                 int64_t pre_stride, int64_t dpre_stride, int cols, uint32_t nvec, uint32_t total, const int* status) {
  grid_dependency_launch();
  grid_dependency_wait();
  const uint32_t idx = blockIdx.x * 256u + threadIdx.x;
  const bool exists = idx < total;
  if (!IN_PLACE && !exists) return;
  const uint32_t row = exists ? idx / nvec : 0u;
  const int col = exists ? (int)(idx - row * nvec) * 8 : cols;
  dh += row * dh_stride + col;
  gate += row * pre_stride + col;
  up += row * pre_stride + col;
  dgate += row * dpre_stride + col;
  dup += row * dpre_stride + col;
  ElemPack<DT, 8> a, g, u, da, db;
  const bool whole = col + 8 <= cols;
  if (whole) {
    a.raw = *reinterpret_cast<const uint4*>(dh);
    g.raw = *reinterpret_cast<const uint4*>(gate);
    u.raw = *reinterpret_cast<const uint4*>(up);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool in = col + i < cols;
      a.h[i] = in ? dh[i] : (uint16_t)0;
      g.h[i] = in ? gate[i] : (uint16_t)0;
      u.h[i] = in ? up[i] : (uint16_t)0;
    }
  }
  if (IN_PLACE && cta_should_skip(status)) return;
  float x[8], y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 v = activate_grad<ACT>(g.get(i));
    x[i] = a.get(i) * u.get(i) * v.y;
    y[i] = a.get(i) * v.x;
  }
  da.set(x);
  db.set(y);
  if (whole) {
    *reinterpret_cast<uint4*>(dgate) = da.raw;
    *reinterpret_cast<uint4*>(dup) = db.raw;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + i < cols) { dgate[i] = da.h[i]; dup[i] = db.h[i]; }
  }
}

template <int DT, bool IN_PLACE>
static cudaError_t launch_gate_grad(const cfk_ffn_gated_backward_args* a, const int* status, cudaStream_t st) {
  const int64_t dh_s = packed(a->dh_stride, a->n), pre_s = packed(a->pre_stride, a->n), dpre_s = packed(a->dpre_stride, a->n);
  const uint32_t nvec = (uint32_t)((a->n + 7) / 8), total = (uint32_t)a->m * nvec;
  auto kern = a->activation == CFK_ACT_SILU ? gate_grad_kernel<DT, CFK_ACT_SILU, IN_PLACE>
              : a->activation == CFK_ACT_GELU ? gate_grad_kernel<DT, CFK_ACT_GELU, IN_PLACE>
              : a->activation == CFK_ACT_GELU_TANH ? gate_grad_kernel<DT, CFK_ACT_GELU_TANH, IN_PLACE>
                                                   : gate_grad_kernel<DT, CFK_ACT_RELU, IN_PLACE>;
  return launch_overlapped(kern, dim3((total + 255u) / 256u), dim3(256), 0, st, (const uint16_t*)a->dh, (const uint16_t*)a->gate,
                           (const uint16_t*)a->up, (uint16_t*)a->dgate, (uint16_t*)a->dup, dh_s, pre_s, dpre_s, a->n, nvec, total,
                           status);
}

// ---- cuts -------------------------------------------------------------------------------------------------------------------
// Which kernel and which tiles follows from estimates of its time, in us.  Their constants are coefficients of terms that overlap, not
// rates that a part of the chip reaches: fits (root mean square error 8 to 15 %) to a sweep of 1170 calls, 1 to 16000 tokens and
// widths 128 to 16384 and 8192, from before tiles of 48, 96 and 192 tokens existed.  With those, over 1440 calls of 1 to 3000 tokens x all
// cuts that now exist, the cut they choose is slower than the best one measured by 0.5 % (dw) to 2.8 % (8-bit products) on average over
// the calls of a kind, and by 38 % at worst (45 % in a backward call of 88 tokens, where dx went to the kernel for few).
constexpr int kPairs = kSMs / 2;

static bool is_gated(int mode) { return mode == kGated16 || mode == kGatedI8; }
static int k_blocks(int mode, int reduce) {
  const int kb = mode == kProductI8 || mode == kGatedI8 ? 128 : 64;
  return (reduce + kb - 1) / kb;
}

// Three things that run beside each other take the longest one's time and some of the others'.
static float overlapped(float a, float b, float c, float beside) {
  const float most = fmaxf(a, fmaxf(b, c));
  return most + beside * (a + b + c - most);
}

// Clusters of 1, 2, 3, 4, 6 and 8 CTAs that are resident at once, with one and with two CTAs per SM, as
// cudaOccupancyMaxActiveClusters answers on B200.
constexpr int kSplits[6] = {1, 2, 3, 4, 6, 8};
constexpr int kResident[2][6] = {{148, 74, 45, 33, 22, 15}, {296, 148, 93, 71, 45, 33}};

// The kernel for few tokens: what a CTA takes for its k-blocks (a round of the ring, or what an SM takes in), the tiles' traffic
// from L2 and the weights' from DRAM run beside each other; then the epilogue, the exchange of a split, and a start that grows with
// the CTAs where two share an SM.  One CTA per SM with the deepest ring where the clusters fit that way: one gated token of
// 11264 x 4096 bf16 32.0 us against 36.2 with half of it.
struct FewCost {
  float start, crowd, round, intake, l2, dram, beside, column, exchange, per_column, per_part, wave;   // us; KB and bytes per us
};
static float plan_few(int mode, int rows, int cols, int reduce, FewPlan* best) {
  static const FewCost kCost[2] = {{2.5f, 0.33f, 0.166f, 167.f, 18.3e6f, 6.95e6f, 0.23f, 0.02f, 1.8f, 0.023f, 0.045f, 1.7f},
                                   {2.5f, 0.8f, 0.242f, 149.f, 15.9e6f, 8e6f, 0.4f, 0.012f, 0.8f, 0.023f, 0.135f, 0.8f}};
  const FewCost& c = kCost[mode == kGrad];
  const int nw = few_weights(mode), nkb = k_blocks(mode, reduce) * (mode == kGrad ? 2 : 1);
  const int tiles_ch = (cols + 127) / 128;
  float best_t = 0.f;
  static const int kTokens[8] = {16, 32, 48, 64, 96, 128, 192, 256};
  for (int j = 0; j < 8 && kTokens[j] <= 256 / nw && (j == 0 || kTokens[j - 1] < rows); ++j) {
    const int tt = kTokens[j];
    const int stage = nw * 16384 + tt * 128, half = (kFewSmemHalf - kFewHead) / stage, full = (kFewSmemFull - kFewHead) / stage;
    const int tiles_tok = (rows + tt - 1) / tt, ntok = rows < tt ? rows : tt;
    const long long tiles = (long long)tiles_ch * tiles_tok;
    if (tiles > 65536) continue;
    const float l2 = (float)tiles * (float)nkb * (float)stage / c.l2;
    const float dram = (float)tiles_ch * (float)nkb * (float)(nw * 16384) / c.dram;
    for (int i = 0; i < 6; ++i) {
      const int s = kSplits[i];
      if (s > nkb) break;
      const bool two = half >= 3 && tiles > kResident[0][i];
      const int resident = kResident[two][i], waves = (int)((tiles + resident - 1) / resident);
      const float live = (float)((tiles < resident ? (int)tiles : resident) * s) / (float)kSMs;     // CTAs per SM
      const float chain = (float)(waves * ((nkb + s - 1) / s)) *
                          fmaxf(c.round, (two && live > 1.f ? live : 1.f) * (float)stage / 1024.f / c.intake);
      const float finish = c.column * (float)(nw * ntok) / (float)s +
                           (s > 1 ? c.exchange + c.per_column * (float)(nw * ntok) + c.per_part * (float)s : 0.f);
      const float t = c.start + (two ? c.crowd * live : 0.f) + overlapped(chain, l2, dram, c.beside) + finish +
                      (float)(waves - 1) * (c.wave + finish);
      if (best_t == 0.f || t < best_t) {
        const int stages = two ? half : full;
        best_t = t;
        *best = FewPlan{tt, s, stages < kFewMaxStages ? stages : kFewMaxStages, tiles_ch, tiles_tok};
      }
    }
  }
  return best_t;
}

static long long set_width(PairJob* j, bool gated, int bn) {
  j->bn = bn;
  j->tiles_r = (j->rows + 255) / 256;
  j->tiles_c = (j->cols + (gated ? bn : 2 * bn) - 1) / (gated ? bn : 2 * bn);
  return (long long)j->tiles_r * j->tiles_c * j->batches;
}
// Widths of the tiles of a launch on CTA pairs, and how the pairs share two lists of them.  MN-major k-blocks of narrow tiles take
// nearly as long as of wide ones (four loads of 64 x 64).  The gradients of 12158 tokens of 768 x 1472 take 108 us; with the second list
// dealt to all pairs alike, whatever they had of the first, 171.
static float plan_pairs(int mode, PairPlan* plan) {
  static const int kWidth[3] = {128, 96, 64};
  static const float kBlock[2][3] = {{0.276f, 0.207f, 0.166f}, {0.27f, 0.235f, 0.20f}};
  const bool gated = is_gated(mode);
  PairPlan best = *plan;
  float best_t = 0.f;
  for (int w = 0; w < (plan->jobs > 1 ? 9 : 3); ++w) {
    const int width[2] = {w % 3, w / 3};
    long long tiles[2] = {0, 0};
    float each[2] = {0.f, 0.f}, last[2] = {0.f, 0.f}, l2 = 0.f, dram = 0.f;      // last two: bytes
    for (int i = 0; i < plan->jobs; ++i) {
      PairJob& j = plan->job[i];
      const int bn = kWidth[width[i]], nkb = k_blocks(mode, j.reduce) * (mode == kGrad && j.kind == 0 ? 2 : 1);
      tiles[i] = set_width(&j, gated, bn);
      last[i] = 1.3f * (float)bn / 128.f;
      each[i] = 1.f + fmaxf((float)nkb * kBlock[mode == kGrad][width[i]], last[i]);
      l2 += (float)tiles[i] * (float)nkb * (float)(32768 + 2 * bn * 128);
      dram += (float)nkb * 128.f * ((float)j.tiles_r * 256.f + (float)j.tiles_c * (float)(2 * bn)) * (float)j.batches;
    }
    const long long all = tiles[0] + tiles[1], pairs = all < kPairs ? all : kPairs;
    const long long most = tiles[0] / pairs, more = tiles[0] % pairs;      // `more` pairs have most + 1 tiles of the first list
    long long share = 0;
    float longest = (float)(most + (more > 0)) * each[0] + last[0];
    if (tiles[1] > 0) {
      // the least that leaves the other pairs no later than those with one tile more, or one less than that
      const float even = ((float)tiles[1] * each[1] - (float)(pairs - more) * each[0]) / ((float)pairs * each[1]);
      const long long from = even > 0.f ? (long long)even : 0, limit = more > 0 ? tiles[1] / more : 0;
      longest = 0.f;
      for (long long x = from; x <= from + 1; ++x) {
        const long long s = x < limit ? x : limit, rest = tiles[1] - more * s, others = (rest + pairs - more - 1) / (pairs - more);
        const float a = more > 0 ? (float)(most + 1) * each[0] + (float)s * each[1] + (s > 0 ? last[1] : last[0]) : 0.f;
        const float b = (float)most * each[0] + (float)others * each[1] + (others > 0 ? last[1] : last[0]);
        if (longest == 0.f || fmaxf(a, b) < longest) { longest = fmaxf(a, b); share = s; }
      }
    }
    const float t = 3.f + overlapped(longest, l2 / 17e6f, dram / (mode == kGrad ? 3.2e6f : 6.3e6f), 0.22f);
    if (best_t == 0.f || t < best_t) {
      best_t = t;
      best = *plan;
      best.pairs = (int)pairs;
      best.share = (int)share;
    }
  }
  *plan = best;
  return best_t;
}
static bool too_many_tiles(const PairPlan& plan) {
  long long n = 0;
  for (int i = 0; i < plan.jobs; ++i) n += (long long)plan.job[i].tiles_r * plan.job[i].tiles_c * plan.job[i].batches;
  return n > 0x7fffffffLL - kPairs;
}

// A forward product: few.tt = 0, or the pairs are not used.
struct ProductPlan { FewPlan few; PairPlan pair; };
static ProductPlan plan_product(int mode, int rows, int cols, int reduce) {
  ProductPlan plan;
  std::memset(&plan, 0, sizeof(plan));
  plan.pair.jobs = 1;
  PairJob& j = plan.pair.job[0];
  j.rows = rows; j.cols = cols; j.reduce = reduce; j.batches = 1;
  const float few = plan_few(mode, rows, cols, reduce, &plan.few), pair = plan_pairs(mode, &plan.pair);
  if (few == 0.f || pair < few) plan.few.tt = 0;
  return plan;
}
// The backward products: dx in the kernel for few tokens (few.tt > 0) or on pairs, there in one launch with the weights' gradients.
static ProductPlan plan_backward(const cfk_ffn_gated_backward_args* a) {
  ProductPlan plan;
  std::memset(&plan, 0, sizeof(plan));
  PairJob dx, dw;
  std::memset(&dx, 0, sizeof(dx));
  dw = dx;
  dx.rows = a->m; dx.cols = a->k; dx.reduce = a->n; dx.batches = 1;
  dw.kind = 1; dw.rows = a->n; dw.cols = a->k; dw.reduce = a->m; dw.batches = 2;
  PairPlan alone = plan.pair, both = plan.pair;
  float t_alone = 0.f;
  if (a->dw_gate) {
    alone.jobs = 1;
    alone.job[0] = dw;
    t_alone = plan_pairs(kGrad, &alone);
  }
  plan.pair = alone;
  if (!a->dx) return plan;
  both.jobs = a->dw_gate ? 2 : 1;
  both.job[0] = dx;
  both.job[1] = dw;
  if (both.jobs == 2 && k_blocks(kGrad, a->m) > 2 * k_blocks(kGrad, a->n)) std::swap(both.job[0], both.job[1]);   // longest tiles first
  const float few = plan_few(kGrad, a->m, a->k, a->n, &plan.few), t_both = plan_pairs(kGrad, &both);
  if (few == 0.f || t_both < few + t_alone) {
    plan.few.tt = 0;
    plan.pair = both;
  }
  return plan;
}

// ---- descriptors ------------------------------------------------------------------------------------------------------------
struct Matrix {
  const void* base;
  int dtype, rows, cols;
  int64_t stride;
};
static bool rows_ok(const Matrix& m) { return rows_ok(m.base, m.dtype, m.cols, m.stride); }
// Read in boxes of 128 bytes x `box_rows` rows.
static int encode(CUtensorMap* map, const Matrix& m, int box_rows) {
  const uint64_t esz = (uint64_t)dtype_size(m.dtype);
  const uint64_t dims[3] = {(uint64_t)m.cols, (uint64_t)m.rows, 1};
  const uint64_t strides[2] = {(uint64_t)m.stride * esz, (uint64_t)m.stride * esz};
  const uint32_t box[3] = {(uint32_t)(128 / esz), (uint32_t)box_rows, 1};
  return encode_tiled(map, m.dtype, 3, m.base, dims, strides, box, 128);
}

// Operands and results as in ProductMaps and ProductParams; unused ones have a null base.
struct ProductCall {
  Matrix x[2], y[3], d[3];
  Matrix elementwise[3];      // what the elementwise launch of the backward pass reads: dh, gate, up
  ProductParams p;
};

// No result shares memory with another or with what the call reads, but for a result of the elementwise launch in the very place of its
// input.
static bool results_apart(const ProductCall& c, bool backward) {
  const auto span = [](const Matrix& m) {
    const int64_t e = dtype_size(m.dtype);
    return RowSpan{m.base, m.rows, m.cols * e, m.stride * e};
  };
  const auto vec = [](const float* v, int n) { return RowSpan{v, 1, 4 * (int64_t)n, 4 * (int64_t)n}; };
  RowSpan out[5], in[8];
  int outs = 0, ins = 0;
  for (const Matrix& m : c.d) out[outs++] = span(m);
  for (const Matrix& m : c.y) in[ins++] = span(m);
  if (backward) {
    for (const Matrix& m : c.x) out[outs++] = span(m);               // dgate, dup
    in[ins++] = span(c.elementwise[0]);
    for (int i = 0; i < 2; ++i)
      if (c.elementwise[1 + i].base != c.x[i].base) in[ins++] = span(c.elementwise[1 + i]);
  } else {
    in[ins++] = span(c.x[0]);
    in[ins++] = vec(c.p.row_scale, c.p.rows);
    for (const float* v : {c.p.col_scale, c.p.col_scale2, c.p.bias}) in[ins++] = vec(v, c.p.cols);
  }
  for (int i = 0; i < outs; ++i) {
    for (int j = 0; j < i; ++j)
      if (share_memory(out[i], out[j])) return false;
    for (int j = 0; j < ins; ++j)
      if (share_memory(out[i], in[j])) return false;
  }
  return true;
}

static int prepare_results(const ProductCall& c, ProductParams* p) {
  int rc = CFK_OK;
  p->status = device_status_block(&rc);
  p->wide = 1;
  for (int i = 0; i < 3; ++i) {
    p->d[i] = const_cast<void*>(c.d[i].base);
    p->d_stride[i] = c.d[i].stride;
    if (p->d[i] && (((uintptr_t)p->d[i] | (uintptr_t)(c.d[i].stride * dtype_size(c.d[i].dtype))) & 31u)) p->wide = 0;
  }
  return rc;
}

// All that can fail ahead of a launch: a call of several launches prepares every one before the first.
struct FewLaunch { ProductMaps maps; ProductParams p; FewPlan plan; };
struct PairLaunch { ProductMaps maps; ProductParams p; PairPlan plan; };

template <int MODE>
static int prepare_few(const ProductCall& c, const FewPlan& few, FewLaunch* l) {
  l->p = c.p;
  l->p.acc_limit = kWaitLimitNs + kNsPerBlock * (unsigned long long)(k_blocks(MODE, c.p.reduce) * (MODE == kGrad ? 2 : 1));
  l->plan = few;
  std::memset(&l->maps, 0, sizeof(l->maps));
  int rc = prepare_results(c, &l->p);
  for (int i = 0; i < 2 && rc == CFK_OK; ++i) {
    if (c.x[i].base) rc = encode(&l->maps.x[i], c.x[i], few.tt);
    if (rc == CFK_OK && c.y[i].base) rc = encode(&l->maps.y[i], c.y[i], MODE == kGrad ? 64 : 128);
  }
  return rc ? rc : allow_few_product<MODE>();
}

template <int MODE>
static int prepare_pairs(const ProductCall& c, PairPlan plan, PairLaunch* l) {
  const int first = plan.job[0].tiles_r * plan.job[0].tiles_c * plan.job[0].batches;
  plan.most = first / plan.pairs;
  plan.more = first % plan.pairs;
  plan.staged = MODE == kGrad && plan.job[plan.jobs - 1].kind == 1 && plan.job[plan.jobs - 1].reduce <= 512;   // weights' gradients
  for (int i = 0; i < plan.jobs; ++i) {
    PairJob& j = plan.job[i];
    j.per_batch = make_divisor((uint32_t)(j.tiles_r * j.tiles_c));
    j.per_band = make_divisor((uint32_t)(kGemmBand * j.tiles_c));
    j.tail_rows = make_divisor((uint32_t)(j.tiles_r % kGemmBand ? j.tiles_r % kGemmBand : 1));
  }
  int longest = 0;                   // k-blocks of a tile
  for (int i = 0; i < plan.jobs; ++i) {
    const int n = k_blocks(MODE, plan.job[i].reduce) * (MODE == kGrad && plan.job[i].kind == 0 ? 2 : 1);
    if (n > longest) longest = n;
  }
  l->p = c.p;
  l->p.acc_limit = kWaitLimitNs + kNsPerBlock * (unsigned long long)longest;
  l->plan = plan;
  std::memset(&l->maps, 0, sizeof(l->maps));
  int rc = prepare_results(c, &l->p);
  for (int i = 0; i < 2 && rc == CFK_OK; ++i)
    if (c.x[i].base) rc = encode(&l->maps.x[i], c.x[i], MODE == kGrad ? 64 : 128);
  for (int i = 0; i < 3 && rc == CFK_OK; ++i)
    if (c.y[i].base) rc = encode(&l->maps.y[i], c.y[i], MODE == kGrad ? 64 : plan.job[0].bn);
  return rc ? rc : allow_pair_product<MODE>();
}

template <int MODE>
static int run_product(const ProductCall& c, cudaStream_t stream) {
  const ProductPlan plan = plan_product(MODE, c.p.rows, c.p.cols, c.p.reduce);
  if (plan.few.tt == 0 && too_many_tiles(plan.pair)) return CFK_ERR_UNSUPPORTED;
  if (!results_apart(c, false)) return CFK_ERR_INVALID_ARG;
  if (plan.few.tt > 0) {
    FewLaunch l;
    const int rc = prepare_few<MODE>(c, plan.few, &l);
    return rc ? rc : launch_few_product<MODE>(l.maps, l.p, l.plan, stream);
  }
  PairLaunch l;
  const int rc = prepare_pairs<MODE>(c, plan.pair, &l);
  return rc ? rc : launch_pair_product<MODE>(l.maps, l.p, l.plan, stream);
}

constexpr int kMaxSize = 0x7fffff00;
static bool is16(int dt) { return dt == CFK_FP16 || dt == CFK_BF16; }
static bool floats_ok(const float* p) { return p != nullptr && ((uintptr_t)p & 3u) == 0; }

// Sizes that can be rounded up to a tile in 32 bits
static bool size_ok(int m, int n, int k) { return m <= kMaxSize && n <= kMaxSize && k <= kMaxSize; }

// 32-bit sums of 8-bit products: k * 128 * 128 stays below 2^31
constexpr int kMaxI8Reduction = 131071;

// Argument checks of the three calls; what passes is ready to be cut and run.
static int check_gemm_i8(const cfk_gemm_i8_args* a, ProductCall* c) {
  if (!a || !a->a || !a->b || !a->c || a->m <= 0 || a->n <= 0 || a->k <= 0) return CFK_ERR_INVALID_ARG;
  if (!is16(a->out_dtype) && a->out_dtype != CFK_FP32) return CFK_ERR_INVALID_ARG;
  if (!floats_ok(a->a_scale) || !floats_ok(a->b_scale) || ((uintptr_t)a->bias & 3u)) return CFK_ERR_INVALID_ARG;
  std::memset(c, 0, sizeof(*c));
  c->x[0] = {a->a, CFK_INT8, a->m, a->k, packed(a->a_stride, a->k)};
  c->y[0] = {a->b, CFK_INT8, a->n, a->k, packed(a->b_stride, a->k)};
  c->d[0] = {a->c, a->out_dtype, a->m, a->n, packed(a->c_stride, a->n)};
  if (!rows_ok(c->x[0]) || !rows_ok(c->y[0]) || !rows_ok(c->d[0])) return CFK_ERR_INVALID_ARG;
  if (a->k > kMaxI8Reduction || !size_ok(a->m, a->n, a->k)) return CFK_ERR_UNSUPPORTED;
  c->p.rows = a->m; c->p.cols = a->n; c->p.reduce = a->k;
  c->p.out = a->out_dtype;
  c->p.row_scale = a->a_scale; c->p.col_scale = a->b_scale; c->p.bias = a->bias;
  return CFK_OK;
}

static int check_gated(const cfk_ffn_gated_args* a, ProductCall* c) {
  if (!a || !a->x || !a->w_gate || !a->w_up || !a->h || a->m <= 0 || a->n <= 0 || a->k <= 0) return CFK_ERR_INVALID_ARG;
  const bool i8 = a->dtype == CFK_INT8;
  if ((!is16(a->dtype) && !i8) || !is16(a->out_dtype) || (!i8 && a->out_dtype != a->dtype)) return CFK_ERR_INVALID_ARG;
  if (a->activation < CFK_ACT_SILU || a->activation > CFK_ACT_RELU) return CFK_ERR_INVALID_ARG;
  if ((a->gate == nullptr) != (a->up == nullptr)) return CFK_ERR_INVALID_ARG;
  if (i8 ? !floats_ok(a->x_scale) || !floats_ok(a->gate_scale) || !floats_ok(a->up_scale)
         : a->x_scale || a->gate_scale || a->up_scale)
    return CFK_ERR_INVALID_ARG;
  std::memset(c, 0, sizeof(*c));
  const int64_t w_stride = packed(a->w_stride, a->k), pre_stride = packed(a->pre_stride, a->n);
  c->x[0] = {a->x, a->dtype, a->m, a->k, packed(a->x_stride, a->k)};
  c->y[0] = {a->w_gate, a->dtype, a->n, a->k, w_stride};
  c->y[1] = {a->w_up, a->dtype, a->n, a->k, w_stride};
  c->d[0] = {a->h, a->out_dtype, a->m, a->n, packed(a->h_stride, a->n)};
  if (a->gate) {
    c->d[1] = {a->gate, a->out_dtype, a->m, a->n, pre_stride};
    c->d[2] = {a->up, a->out_dtype, a->m, a->n, pre_stride};
    if (!rows_ok(c->d[1]) || !rows_ok(c->d[2])) return CFK_ERR_INVALID_ARG;
    if (a->gate == a->up || a->gate == a->h || a->up == a->h) return CFK_ERR_INVALID_ARG;
  }
  if (!rows_ok(c->x[0]) || !rows_ok(c->y[0]) || !rows_ok(c->y[1]) || !rows_ok(c->d[0])) return CFK_ERR_INVALID_ARG;
  if ((i8 && a->k > kMaxI8Reduction) || !size_ok(a->m, a->n, a->k)) return CFK_ERR_UNSUPPORTED;
  c->p.rows = a->m; c->p.cols = a->n; c->p.reduce = a->k;
  c->p.bf16 = a->dtype == CFK_BF16; c->p.out = a->out_dtype;
  c->p.act = a->activation; c->p.keep = a->gate != nullptr;
  c->p.row_scale = a->x_scale; c->p.col_scale = a->gate_scale; c->p.col_scale2 = a->up_scale;
  return CFK_OK;
}

static int check_backward(const cfk_ffn_gated_backward_args* a, ProductCall* c) {
  if (!a || !a->dh || !a->x || !a->w_gate || !a->w_up || !a->gate || !a->up || !a->dgate || !a->dup) return CFK_ERR_INVALID_ARG;
  if (a->m <= 0 || a->n <= 0 || a->k <= 0 || !is16(a->dtype)) return CFK_ERR_INVALID_ARG;
  if (a->activation < CFK_ACT_SILU || a->activation > CFK_ACT_RELU) return CFK_ERR_INVALID_ARG;
  if ((a->dw_gate == nullptr) != (a->dw_up == nullptr)) return CFK_ERR_INVALID_ARG;
  const int dt = a->dtype;
  const int64_t pre_s = packed(a->pre_stride, a->n), dpre_s = packed(a->dpre_stride, a->n);
  const int64_t w_s = packed(a->w_stride, a->k), dw_s = packed(a->dw_stride, a->k);
  std::memset(c, 0, sizeof(*c));
  c->x[0] = {a->dgate, dt, a->m, a->n, dpre_s};
  c->x[1] = {a->dup, dt, a->m, a->n, dpre_s};
  c->y[0] = {a->w_gate, dt, a->n, a->k, w_s};
  c->y[1] = {a->w_up, dt, a->n, a->k, w_s};
  c->y[2] = {a->x, dt, a->m, a->k, packed(a->x_stride, a->k)};
  c->d[0] = {a->dx, dt, a->m, a->k, packed(a->dx_stride, a->k)};
  c->d[1] = {a->dw_gate, dt, a->n, a->k, dw_s};
  c->d[2] = {a->dw_up, dt, a->n, a->k, dw_s};
  Matrix* const in = c->elementwise;
  in[0] = {a->dh, dt, a->m, a->n, packed(a->dh_stride, a->n)};
  in[1] = {a->gate, dt, a->m, a->n, pre_s};
  in[2] = {a->up, dt, a->m, a->n, pre_s};
  for (int i = 0; i < 3; ++i)
    if (!rows_ok(in[i]) || !rows_ok(c->y[i]) || (i < 2 && !rows_ok(c->x[i])) || (c->d[i].base && !rows_ok(c->d[i])))
      return CFK_ERR_INVALID_ARG;
  // dgate may take the place of gate and dup that of up, row for row (results_apart has the rest)
  if (a->dgate == a->dup || a->dgate == a->up || a->dup == a->gate || a->dgate == a->dh || a->dup == a->dh) return CFK_ERR_INVALID_ARG;
  if ((a->dgate == a->gate || a->dup == a->up) && pre_s != dpre_s) return CFK_ERR_INVALID_ARG;
  if (!size_ok(a->m, a->n, a->k) || (long long)a->m * ((a->n + 7) / 8) > 0xffffff00LL) return CFK_ERR_UNSUPPORTED;
  c->p.rows = a->m; c->p.cols = a->k; c->p.reduce = a->n;
  c->p.bf16 = dt == CFK_BF16; c->p.out = dt;
  return CFK_OK;
}

static int tell_plan(int rc, int mode, const ProductCall& c, int plan[3]) {
  if (rc != CFK_OK || !plan) return rc != CFK_OK ? rc : CFK_ERR_INVALID_ARG;
  const ProductPlan p = plan_product(mode, c.p.rows, c.p.cols, c.p.reduce);
  plan[0] = p.few.tt > 0; plan[1] = p.few.tt > 0 ? p.few.tt : p.pair.job[0].bn; plan[2] = p.few.tt > 0 ? p.few.splits : 1;
  return CFK_OK;
}

}  // namespace cfk

using namespace cfk;

extern "C" int cfk_gemm_i8(const cfk_gemm_i8_args* a, cfk_stream_t stream) {
  ProductCall c;
  const int rc = check_gemm_i8(a, &c);
  return rc ? rc : run_product<kProductI8>(c, (cudaStream_t)stream);
}
extern "C" int cfk_gemm_i8_plan(const cfk_gemm_i8_args* a, int plan[3]) {
  ProductCall c;
  const int rc = check_gemm_i8(a, &c);
  return tell_plan(rc, kProductI8, c, plan);
}

extern "C" int cfk_ffn_gated(const cfk_ffn_gated_args* a, cfk_stream_t stream) {
  ProductCall c;
  const int rc = check_gated(a, &c);
  if (rc) return rc;
  return a->dtype == CFK_INT8 ? run_product<kGatedI8>(c, (cudaStream_t)stream) : run_product<kGated16>(c, (cudaStream_t)stream);
}
extern "C" int cfk_ffn_gated_plan(const cfk_ffn_gated_args* a, int plan[3]) {
  ProductCall c;
  const int rc = check_gated(a, &c);
  return tell_plan(rc, rc == CFK_OK && a->dtype == CFK_INT8 ? kGatedI8 : kGated16, c, plan);
}

extern "C" int cfk_ffn_gated_backward(const cfk_ffn_gated_backward_args* a, cfk_stream_t stream) {
  ProductCall c;
  int rc = check_backward(a, &c);
  if (rc) return rc;
  const ProductPlan plan = plan_backward(a);
  if (too_many_tiles(plan.pair)) return CFK_ERR_UNSUPPORTED;
  if (!results_apart(c, true)) return CFK_ERR_INVALID_ARG;
  const int* status = device_status_block(&rc);
  if (!status) return rc;
  // in place the first launch takes the place of its inputs: nothing that could fail is left for after it but the launches
  FewLaunch few;
  PairLaunch pair;
  if (plan.few.tt > 0 && (rc = prepare_few<kGrad>(c, plan.few, &few))) return rc;
  if (plan.pair.jobs > 0 && (rc = prepare_pairs<kGrad>(c, plan.pair, &pair))) return rc;
  const cudaStream_t st = (cudaStream_t)stream;
  const bool in_place = a->dgate == a->gate || a->dup == a->up;
  const auto launch = a->dtype == CFK_FP16 ? (in_place ? launch_gate_grad<CFK_FP16, true> : launch_gate_grad<CFK_FP16, false>)
                                           : (in_place ? launch_gate_grad<CFK_BF16, true> : launch_gate_grad<CFK_BF16, false>);
  if (note_cuda(launch(a, status, st), "gate gradient launch") != cudaSuccess) return CFK_ERR_LAUNCH;
  if (plan.few.tt > 0 && (rc = launch_few_product<kGrad>(few.maps, few.p, few.plan, st))) return rc;
  return plan.pair.jobs > 0 ? launch_pair_product<kGrad>(pair.maps, pair.p, pair.plan, st) : CFK_OK;
}
extern "C" int cfk_ffn_gated_backward_plan(const cfk_ffn_gated_backward_args* a, int plan[4]) {
  ProductCall c;
  const int rc = check_backward(a, &c);
  if (rc != CFK_OK || !plan) return rc != CFK_OK ? rc : CFK_ERR_INVALID_ARG;
  const ProductPlan p = plan_backward(a);
  plan[0] = p.few.tt > 0; plan[1] = p.few.tt; plan[2] = p.few.tt > 0 ? p.few.splits : 1; plan[3] = 0;
  for (int i = 0; i < p.pair.jobs; ++i) plan[p.pair.job[i].kind == 0 ? 1 : 3] = p.pair.job[i].bn;
  return CFK_OK;
}
