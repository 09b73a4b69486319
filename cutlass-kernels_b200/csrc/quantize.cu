// cfk_quantize_rows: symmetric 8-bit quantisation with a scale per row (include/cfk_b200.h has the definition).
#include "common.cuh"
#include "element_io.cuh"
#include "host_util.h"

namespace cfk {

// Memory bound: each element is read once and written once as a byte, so a row is held in registers between the maximum and
// the rounding.  G threads share a row and hold up to 8 vectors of 8 elements each; of a row longer than that (16384 elements
// with 256 threads) the rest is read a second time, from L2.
//
// The maximum is taken on the bit patterns of |x|, which order like the values and put infinity and NaN on top, so that one
// comparison afterwards finds a row that holds either.
//
// q is defined by a division rounded to fp32 and a rounding to an integer.  The product with 1 / scale differs from that quotient by
// less than 1e-4 (|q| <= 127, three roundings of 2^-24 each), so both round to the same integer unless the product
// lies within 1e-4 of the middle between two; only then is the division made.
constexpr float kTieDistance = 1e-4f;

__device__ __forceinline__ float quantize_one(float x, float scale, float inv) {
  const float t = x * inv;
  float r = rintf(t);
  if (!(fabsf(t - r) <= 0.5f - kTieDistance)) r = rintf(__fdiv_rn(x, scale));   // also where inv overflowed
  return fminf(fmaxf(r, -127.f), 127.f);
}

template <int SDT, int G>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const void* src, int64_t src_stride, int8_t* dst,
                                                            int64_t dst_stride, float* scale, int rows, int cols) {
  constexpr int U = 8, PER = 256 / G, SB = elem_bytes(SDT);
  using Half = ElemPack<SDT, 16 / SB>;           // one 16-byte access: 8 elements, or 4 of fp32
  constexpr int NH = 8 / (16 / SB);              // accesses per vector of 8
  __shared__ uint32_t s_max[8];
  grid_dependency_launch();
  grid_dependency_wait();
  const int t = threadIdx.x % G;
  const int64_t row = (int64_t)blockIdx.x * PER + threadIdx.x / G;
  if (G == 32 && row >= rows) return;            // a whole warp; with G = 256 every block has a row
  const char* s = reinterpret_cast<const char*>(src) + row * src_stride * SB;
  int8_t* d = dst + row * dst_stride;
  const int nvec = (cols + 7) / 8;

  auto load = [&](int v, float (&x)[8]) {        // elements 8 v .. 8 v + 7; those behind the row's end read as 0
    if (v * 8 + 8 <= cols) {
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        Half p;
        p.raw = __ldg(reinterpret_cast<const uint4*>(s + (int64_t)v * 8 * SB) + h);
#pragma unroll
        for (int i = 0; i < 16 / SB; ++i) x[h * (16 / SB) + i] = p.get(i);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = 0.f;
        if (v * 8 + i < cols) {
          ElemPack<SDT, 1> e;
          e.raw = reinterpret_cast<const typename RawBytes<SB>::type*>(s)[(int64_t)v * 8 + i];
          x[i] = e.get(0);
        }
      }
    }
  };

  float x[U][8];
  uint32_t m = 0u;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (t + u * G < nvec) {
      load(t + u * G, x[u]);
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[u][i]) & 0x7fffffffu);
    }
  }
  for (int v = t + U * G; v < nvec; v += G) {
    float y[8];
    load(v, y);
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(y[i]) & 0x7fffffffu);
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if (G > 32) {
    if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < G / 32; ++w) m = max(m, s_max[w]);
  }
  const bool finite = m < 0x7f800000u;
  const float sc = finite ? __fdiv_rn(__uint_as_float(m), 127.f) : __uint_as_float(0x7fffffffu);
  if (t == 0) scale[row] = sc;
  const bool zero = !finite || sc == 0.f;
  const float inv = zero ? 0.f : __fdiv_rn(1.f, sc);

  auto store = [&](int v, const float (&y)[8]) {
    uint32_t w[2] = {0u, 0u};
    if (!zero) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        w[i >> 2] |= ((uint32_t)(int)quantize_one(y[i], sc, inv) & 0xffu) << (8 * (i & 3));
    }
    if (v * 8 + 8 <= cols) {
      *reinterpret_cast<uint2*>(d + (int64_t)v * 8) = make_uint2(w[0], w[1]);
    } else {
      for (int i = 0; v * 8 + i < cols; ++i) d[(int64_t)v * 8 + i] = (int8_t)(w[i >> 2] >> (8 * (i & 3)));
    }
  };
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (t + u * G < nvec) store(t + u * G, x[u]);
  for (int v = t + U * G; v < nvec; v += G) {
    float y[8];
    load(v, y);
    store(v, y);
  }
}

template <int SDT>
static cudaError_t launch_quantize(const void* src, int64_t ss, void* dst, int64_t ds, float* scale, int rows, int cols,
                                   cudaStream_t st) {
  // a warp per row while it can hold the row in a few vectors per thread, else a block per row
  if (cols <= 1024)
    return launch_overlapped(quantize_rows_kernel<SDT, 32>, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, st, src, ss,
                             (int8_t*)dst, ds, scale, rows, cols);
  return launch_overlapped(quantize_rows_kernel<SDT, 256>, dim3((unsigned)rows), dim3(256), 0, st, src, ss, (int8_t*)dst, ds,
                           scale, rows, cols);
}

}  // namespace cfk

using namespace cfk;

extern "C" int cfk_quantize_rows(const void* src, int src_dtype, int64_t src_stride, void* dst, int64_t dst_stride,
                                 float* scale, int rows, int cols, cfk_stream_t stream) {
  if (!src || !dst || !scale || rows <= 0 || cols <= 0) return CFK_ERR_INVALID_ARG;
  if (src_dtype != CFK_FP16 && src_dtype != CFK_BF16 && src_dtype != CFK_FP32) return CFK_ERR_INVALID_ARG;
  if (src_stride == 0) src_stride = cols;
  if (dst_stride == 0) dst_stride = cols;
  if (!rows_ok(src, src_dtype, cols, src_stride) || !rows_ok(dst, CFK_INT8, cols, dst_stride) || ((uintptr_t)scale & 3u))
    return CFK_ERR_INVALID_ARG;
  const cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e;
  switch (src_dtype) {
    case CFK_FP16: e = launch_quantize<CFK_FP16>(src, src_stride, dst, dst_stride, scale, rows, cols, st); break;
    case CFK_BF16: e = launch_quantize<CFK_BF16>(src, src_stride, dst, dst_stride, scale, rows, cols, st); break;
    default: e = launch_quantize<CFK_FP32>(src, src_stride, dst, dst_stride, scale, rows, cols, st); break;
  }
  return note_cuda(e, "quantize launch") == cudaSuccess ? CFK_OK : CFK_ERR_LAUNCH;
}
