// Entry points of the feed-forward operators (include/cfk_b200.h): argument checks, descriptors and choice of kernel, and the
// elementwise part of the gated block's backward pass.
#include <cstring>

#include "common.cuh"
#include "element_io.cuh"
#include "ffn_act.cuh"
#include "ffn_params.h"
#include "host_util.h"

namespace cfk {

// dgate = dh * up * act'(gate), dup = dh * act(gate).  Memory bound: three 16-bit values in, two out, 16 bytes per access, a thread
// reads its elements of all three before it writes, so the results may take the place of gate and up.
template <int DT, int ACT>
__global__ void __launch_bounds__(256) gate_grad_kernel(const uint16_t* dh, const uint16_t* gate, const uint16_t* up, uint16_t* dgate,
                                                        uint16_t* dup, int64_t dh_stride, int64_t pre_stride,
                                                        int64_t dpre_stride, int cols, uint32_t nvec, uint32_t total) {
  grid_dependency_launch();
  grid_dependency_wait();
  const uint32_t idx = blockIdx.x * 256u + threadIdx.x;
  if (idx >= total) return;
  const uint32_t row = idx / nvec;
  const int col = (int)(idx - row * nvec) * 8;
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

template <int DT>
static cudaError_t launch_gate_grad(const cfk_ffn_gated_backward_args* a, int64_t dh_s, int64_t pre_s, int64_t dpre_s,
                                    cudaStream_t st) {
  const uint32_t nvec = (uint32_t)((a->n + 7) / 8), total = (uint32_t)a->m * nvec;
  auto kern = a->activation == CFK_ACT_SILU ? gate_grad_kernel<DT, CFK_ACT_SILU>
              : a->activation == CFK_ACT_GELU ? gate_grad_kernel<DT, CFK_ACT_GELU>
              : a->activation == CFK_ACT_GELU_TANH ? gate_grad_kernel<DT, CFK_ACT_GELU_TANH> : gate_grad_kernel<DT, CFK_ACT_RELU>;
  return launch_overlapped(kern, dim3((total + 255u) / 256u), dim3(256), 0, st, (const uint16_t*)a->dh, (const uint16_t*)a->gate,
                           (const uint16_t*)a->up, (uint16_t*)a->dgate, (uint16_t*)a->dup, dh_s, pre_s, dpre_s, a->n, nvec, total);
}

// ---- descriptors ------------------------------------------------------------------------------------------------------------
// A matrix of `rows` rows of `cols` elements, read or written in boxes of 128 bytes x `box_rows` rows.
static int encode_rows(CUtensorMap* map, int dtype, const void* base, int rows, int cols, int64_t stride, int box_rows) {
  const uint64_t esz = (uint64_t)dtype_size(dtype);
  const uint64_t dims[3] = {(uint64_t)cols, (uint64_t)rows, 1};
  const uint64_t strides[2] = {(uint64_t)stride * esz, (uint64_t)stride * esz};
  const uint32_t box[3] = {(uint32_t)(128 / esz), (uint32_t)box_rows, 1};
  return encode_tiled(map, dtype, 3, base, dims, strides, box, 128);
}

struct Matrix {
  const void* base;
  int dtype, rows, cols;
  int64_t stride;
};
static int encode(CUtensorMap* map, const Matrix& m, int box_rows) {
  return encode_rows(map, m.dtype, m.base, m.rows, m.cols, m.stride, box_rows);
}

// A product's operands and results as matrices; unused ones have a null base.
struct ProductCall {
  Matrix x[2], y[2], d[3];
  ProductParams p;
};

template <int MODE>
static int run_product(const ProductCall& c, cudaStream_t stream) {
  constexpr bool GATED = MODE == kGated16 || MODE == kGatedI8;
  ProductParams p = c.p;
  int rc = CFK_OK;
  p.status = device_status_block(&rc);
  if (!p.status) return rc;
  ProductMaps maps;
  std::memset(&maps, 0, sizeof(maps));
  // K-major operands land as 128 rows of a k-block, MN-major ones as spans of 64 columns of its 64 rows
  for (int i = 0; i < 2; ++i) {
    if (c.x[i].base && (rc = encode(&maps.x[i], c.x[i], MODE == kGradW ? 64 : 128))) return rc;
    if (c.y[i].base && (rc = encode(&maps.y[i], c.y[i], MODE == kGradX || MODE == kGradW ? 64 : 128))) return rc;
  }
  p.whole = p.cols & ~(16 / dtype_size(p.out) - 1);
  for (int i = 0; i < 3; ++i) {
    if (!c.d[i].base) continue;
    Matrix d = c.d[i];
    d.cols = p.whole;
    if (d.cols > 0 && (rc = encode(&maps.d[i], d, 128))) return rc;
    p.d[i] = const_cast<void*>(d.base);
    p.d_stride[i] = d.stride;
  }
  p.tiles_r = (p.rows + 255) / 256;
  p.tiles_c = GATED ? (p.cols + 127) / 128 : (p.cols + 255) / 256;
  if ((long long)p.tiles_r * p.tiles_c * p.batches > 0x7fffffffLL - 1024) return CFK_ERR_UNSUPPORTED;
  return launch_pair_product<MODE>(maps, p, stream);
}

static int64_t packed(int64_t stride, int cols) { return stride == 0 ? cols : stride; }
static bool is16(int dt) { return dt == CFK_FP16 || dt == CFK_BF16; }
static bool floats_ok(const float* p) { return p != nullptr && ((uintptr_t)p & 3u) == 0; }

// 32-bit sums of 8-bit products: k * 128 * 128 stays below 2^31
constexpr int kMaxI8Reduction = 131071;

}  // namespace cfk

using namespace cfk;

extern "C" int cfk_gemm_i8(const cfk_gemm_i8_args* a, cfk_stream_t stream) {
  if (!a || !a->a || !a->b || !a->c || a->m <= 0 || a->n <= 0 || a->k <= 0) return CFK_ERR_INVALID_ARG;
  if (!is16(a->out_dtype) && a->out_dtype != CFK_FP32) return CFK_ERR_INVALID_ARG;
  if (!floats_ok(a->a_scale) || !floats_ok(a->b_scale) || ((uintptr_t)a->bias & 3u)) return CFK_ERR_INVALID_ARG;
  ProductCall c;
  std::memset(&c, 0, sizeof(c));
  c.x[0] = {a->a, CFK_INT8, a->m, a->k, packed(a->a_stride, a->k)};
  c.y[0] = {a->b, CFK_INT8, a->n, a->k, packed(a->b_stride, a->k)};
  c.d[0] = {a->c, a->out_dtype, a->m, a->n, packed(a->c_stride, a->n)};
  if (!rows_ok(a->a, CFK_INT8, a->k, c.x[0].stride) || !rows_ok(a->b, CFK_INT8, a->k, c.y[0].stride) ||
      !rows_ok(a->c, a->out_dtype, a->n, c.d[0].stride))
    return CFK_ERR_INVALID_ARG;
  if (a->k > kMaxI8Reduction) return CFK_ERR_UNSUPPORTED;
  c.p.rows = a->m; c.p.cols = a->n; c.p.reduce = a->k; c.p.batches = 1;
  c.p.out = a->out_dtype;
  c.p.row_scale = a->a_scale; c.p.col_scale = a->b_scale; c.p.bias = a->bias;
  return run_product<kProductI8>(c, (cudaStream_t)stream);
}

extern "C" int cfk_ffn_gated(const cfk_ffn_gated_args* a, cfk_stream_t stream) {
  if (!a || !a->x || !a->w_gate || !a->w_up || !a->h || a->m <= 0 || a->n <= 0 || a->k <= 0) return CFK_ERR_INVALID_ARG;
  const bool i8 = a->dtype == CFK_INT8;
  if ((!is16(a->dtype) && !i8) || !is16(a->out_dtype) || (!i8 && a->out_dtype != a->dtype)) return CFK_ERR_INVALID_ARG;
  if (a->activation < CFK_ACT_SILU || a->activation > CFK_ACT_RELU) return CFK_ERR_INVALID_ARG;
  if ((a->gate == nullptr) != (a->up == nullptr)) return CFK_ERR_INVALID_ARG;
  if (i8 ? !floats_ok(a->x_scale) || !floats_ok(a->gate_scale) || !floats_ok(a->up_scale)
         : a->x_scale || a->gate_scale || a->up_scale)
    return CFK_ERR_INVALID_ARG;
  ProductCall c;
  std::memset(&c, 0, sizeof(c));
  const int64_t w_stride = packed(a->w_stride, a->k), pre_stride = packed(a->pre_stride, a->n);
  c.x[0] = {a->x, a->dtype, a->m, a->k, packed(a->x_stride, a->k)};
  c.y[0] = {a->w_gate, a->dtype, a->n, a->k, w_stride};
  c.y[1] = {a->w_up, a->dtype, a->n, a->k, w_stride};
  c.d[0] = {a->h, a->out_dtype, a->m, a->n, packed(a->h_stride, a->n)};
  if (a->gate) {
    c.d[1] = {a->gate, a->out_dtype, a->m, a->n, pre_stride};
    c.d[2] = {a->up, a->out_dtype, a->m, a->n, pre_stride};
  }
  if (!rows_ok(a->x, a->dtype, a->k, c.x[0].stride) || !rows_ok(a->w_gate, a->dtype, a->k, w_stride) ||
      !rows_ok(a->w_up, a->dtype, a->k, w_stride) || !rows_ok(a->h, a->out_dtype, a->n, c.d[0].stride))
    return CFK_ERR_INVALID_ARG;
  if (a->gate && (!rows_ok(a->gate, a->out_dtype, a->n, pre_stride) || !rows_ok(a->up, a->out_dtype, a->n, pre_stride)))
    return CFK_ERR_INVALID_ARG;
  if (i8 && a->k > kMaxI8Reduction) return CFK_ERR_UNSUPPORTED;
  c.p.rows = a->m; c.p.cols = a->n; c.p.reduce = a->k; c.p.batches = 1;
  c.p.bf16 = a->dtype == CFK_BF16; c.p.out = a->out_dtype;
  c.p.act = a->activation; c.p.keep = a->gate != nullptr;
  c.p.row_scale = a->x_scale; c.p.col_scale = a->gate_scale; c.p.col_scale2 = a->up_scale;
  return i8 ? run_product<kGatedI8>(c, (cudaStream_t)stream) : run_product<kGated16>(c, (cudaStream_t)stream);
}

extern "C" int cfk_ffn_gated_backward(const cfk_ffn_gated_backward_args* a, cfk_stream_t stream) {
  if (!a || !a->dh || !a->x || !a->w_gate || !a->w_up || !a->gate || !a->up || !a->dgate || !a->dup) return CFK_ERR_INVALID_ARG;
  if (a->m <= 0 || a->n <= 0 || a->k <= 0 || !is16(a->dtype)) return CFK_ERR_INVALID_ARG;
  if (a->activation < CFK_ACT_SILU || a->activation > CFK_ACT_RELU) return CFK_ERR_INVALID_ARG;
  if ((a->dw_gate == nullptr) != (a->dw_up == nullptr)) return CFK_ERR_INVALID_ARG;
  const int dt = a->dtype;
  const int64_t dh_s = packed(a->dh_stride, a->n), x_s = packed(a->x_stride, a->k), w_s = packed(a->w_stride, a->k);
  const int64_t pre_s = packed(a->pre_stride, a->n), dpre_s = packed(a->dpre_stride, a->n);
  const int64_t dx_s = packed(a->dx_stride, a->k), dw_s = packed(a->dw_stride, a->k);
  if (!rows_ok(a->dh, dt, a->n, dh_s) || !rows_ok(a->x, dt, a->k, x_s) || !rows_ok(a->w_gate, dt, a->k, w_s) ||
      !rows_ok(a->w_up, dt, a->k, w_s) || !rows_ok(a->gate, dt, a->n, pre_s) || !rows_ok(a->up, dt, a->n, pre_s) ||
      !rows_ok(a->dgate, dt, a->n, dpre_s) || !rows_ok(a->dup, dt, a->n, dpre_s))
    return CFK_ERR_INVALID_ARG;
  if (a->dx && !rows_ok(a->dx, dt, a->k, dx_s)) return CFK_ERR_INVALID_ARG;
  if (a->dw_gate && (!rows_ok(a->dw_gate, dt, a->k, dw_s) || !rows_ok(a->dw_up, dt, a->k, dw_s))) return CFK_ERR_INVALID_ARG;
  // the only buffers that may be shared: dgate on gate, dup on up, row for row
  if (a->dgate == a->dup || a->dgate == a->up || a->dup == a->gate || a->dgate == a->dh || a->dup == a->dh) return CFK_ERR_INVALID_ARG;
  if ((a->dgate == a->gate || a->dup == a->up) && pre_s != dpre_s) return CFK_ERR_INVALID_ARG;
  if ((long long)a->m * ((a->n + 7) / 8) > 0xffffff00LL) return CFK_ERR_UNSUPPORTED;
  const cudaStream_t st = (cudaStream_t)stream;

  ProductCall gx, gw;
  std::memset(&gx, 0, sizeof(gx));
  const Matrix dgate = {a->dgate, dt, a->m, a->n, dpre_s}, dup = {a->dup, dt, a->m, a->n, dpre_s};
  gx.x[0] = dgate; gx.x[1] = dup;
  gx.p.bf16 = dt == CFK_BF16; gx.p.out = dt;
  gw = gx;
  gx.y[0] = {a->w_gate, dt, a->n, a->k, w_s};
  gx.y[1] = {a->w_up, dt, a->n, a->k, w_s};
  gx.d[0] = {a->dx, dt, a->m, a->k, dx_s};
  gx.p.rows = a->m; gx.p.cols = a->k; gx.p.reduce = a->n; gx.p.batches = 1;
  gw.y[0] = {a->x, dt, a->m, a->k, x_s};
  gw.d[0] = {a->dw_gate, dt, a->n, a->k, dw_s};
  gw.d[1] = {a->dw_up, dt, a->n, a->k, dw_s};
  gw.p.rows = a->n; gw.p.cols = a->k; gw.p.reduce = a->m; gw.p.batches = 2;

  const cudaError_t e = dt == CFK_FP16 ? launch_gate_grad<CFK_FP16>(a, dh_s, pre_s, dpre_s, st)
                                       : launch_gate_grad<CFK_BF16>(a, dh_s, pre_s, dpre_s, st);
  if (note_cuda(e, "gate gradient launch") != cudaSuccess) return CFK_ERR_LAUNCH;
  int rc = CFK_OK;
  if (a->dx && (rc = run_product<kGradX>(gx, st))) return rc;
  if (a->dw_gate) rc = run_product<kGradW>(gw, st);
  return rc;
}
