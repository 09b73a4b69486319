// cfk_quantize_rows: symmetric 8-bit quantisation with a scale per row (include/cfk_b200.h has the definition).
#include "common.cuh"
#include "element_io.cuh"
#include "host_util.h"

namespace cfk {

// Memory bound: each element is read once and written once as a byte, so a row is held in registers, as it was read, between the
// maximum and the rounding.  G threads share a row and hold U vectors of 8 elements each; of a row longer than that (16384
// elements with 256 threads) the rest is read a second time, from L2.
//
// The maximum is taken on the bit patterns of |x|, which order like the values and put infinity and NaN on top, so that one
// comparison afterwards finds a row that holds either.
//
// q is defined by a division rounded to fp32.  With the correctly rounded inverse of the scale, one per row, the quotient
// of an element takes a product and two corrections by its exact remainder: the first leaves less than an ulp, the second
// then rounds correctly (P. Markstein, Computation of elementary functions on the IBM RISC System/6000 processor, 1990).
// Remainders must not underflow, so rows of a scale below 2^-90 divide.  Adding 1.5 * 2^23 rounds to an integer, half to even, and
// leaves it in the low bits.  14 instructions per element in all, 80 % of the issue slots: 8192 x 8192 bf16 in 35 us, 5.8 TB/s; fp32,
// with twice the bytes per element, in 48.5 us, 6.9 TB/s.  (With one product, a comparison against the middle between two integers
// and a division where it is near, 25 instructions and 77 us.)
constexpr float kRound = 12582912.f, kSmallestInverted = 8.0779356694631609e-28f;    // 2^-90

__device__ __forceinline__ float quotient(float x, float scale, float inv) {
  float q = x * inv;
  q = fmaf(fmaf(-q, scale, x), inv, q);
  return fmaf(fmaf(-q, scale, x), inv, q);
}
// Largest |x| of a 16-byte access as a bit pattern, merged into m: two 16-bit values side by side, or fp32.
__device__ __forceinline__ uint32_t max_pattern(uint32_t m, uint4 raw, int elem) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (elem == 2) asm("max.u16x2 %0, %0, %1;" : "+r"(m) : "r"(w[i] & 0x7fff7fffu));
    else m = max(m, w[i] & 0x7fffffffu);
  }
  return m;
}
// Element i of a 16-byte access as fp32, straight from its 32-bit words.
template <int SDT>
__device__ __forceinline__ float element(const uint4& raw, int i) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  if constexpr (SDT == CFK_FP32) return __uint_as_float(w[i]);
  else if constexpr (SDT == CFK_BF16) return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
  else {
    const __half2 h = *reinterpret_cast<const __half2*>(&w[i >> 1]);
    return i & 1 ? __high2float(h) : __low2float(h);
  }
}
__device__ __noinline__ uint32_t quantize_by_division(float x, float scale) {     // quotients by a subnormal scale may pass 127
  return (uint32_t)(int)fminf(fmaxf(rintf(__fdiv_rn(x, scale)), -127.f), 127.f);
}

template <int SDT, int G, int U>
__global__ void __launch_bounds__(256, U > 4 ? 2 : elem_bytes(SDT) == 2 ? 5 : 4)
quantize_rows_kernel(const void* src, int64_t src_stride, int8_t* dst, int64_t dst_stride, float* scale, int rows, int cols) {
  constexpr int PER = 256 / G, SB = elem_bytes(SDT), E = 16 / SB;   // elements per 16-byte access: 8, or 4 of fp32
  constexpr int NH = 8 / E;                                        // accesses per vector of 8
  using Half = ElemPack<SDT, E>;
  __shared__ uint32_t s_max[8];
  grid_dependency_launch();
  grid_dependency_wait();
  const int t = threadIdx.x % G;
  const int64_t row = (int64_t)blockIdx.x * PER + threadIdx.x / G;
  if (row >= rows) return;                       // all threads of a row
  const uint4* s = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(src) + row * src_stride * SB);
  int8_t* d = dst + row * dst_stride;
  const int nvec = cols / 8;                     // whole vectors; the elements behind them are one each for the first threads
  const int last = nvec * 8 + t;
  float tail = 0.f;
  if (t < 8 && last < cols) {
    ElemPack<SDT, 1> e;
    e.raw = reinterpret_cast<const typename RawBytes<SB>::type*>(s)[last];
    tail = e.get(0);
  }

  // all loads ahead of the first use, and none behind a branch
  Half x[U][NH];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      x[u][h].raw = make_uint4(0u, 0u, 0u, 0u);
      if (t + u * G < nvec) x[u][h].raw = __ldcs(s + (t + u * G) * NH + h);
    }
  uint32_t m = 0u;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int h = 0; h < NH; ++h) m = max_pattern(m, x[u][h].raw, SB);
  for (int v = t + U * G; v < nvec; v += G) {
#pragma unroll
    for (int h = 0; h < NH; ++h) m = max_pattern(m, s[v * NH + h], SB);
  }
  if constexpr (SB == 2) {                       // as fp32: the larger of the two
    ElemPack<SDT, 1> e;
    e.raw = (uint16_t)max(m & 0xffffu, m >> 16);
    m = __float_as_uint(e.get(0));
  }
  m = max(m, __float_as_uint(tail) & 0x7fffffffu);
  m = __reduce_max_sync(0xffffffffu, m);
  if constexpr (G > 32) {                        // a barrier for each row of the block
    const int first = (threadIdx.x / G) * (G / 32);
    if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
    named_bar_sync(1 + threadIdx.x / G, G);
#pragma unroll
    for (int w = 0; w < G / 32; ++w) m = max(m, s_max[first + w]);
  }
  const bool finite = m < 0x7f800000u;
  const float sc = finite ? __fdiv_rn(__uint_as_float(m), 127.f) : __uint_as_float(0x7fffffffu);
  if (t == 0) scale[row] = sc;
  const bool zero = !finite || sc == 0.f;
  const bool divide = sc < kSmallestInverted;
  const float inv = zero || divide ? 0.f : __fdiv_rn(1.f, sc);

  auto store = [&](int v, const Half (&y)[NH]) {
    uint32_t b[8];
    if (!divide) {
#pragma unroll
      for (int i = 0; i < 8; ++i) b[i] = __float_as_uint(quotient(element<SDT>(y[i / E].raw, i % E), sc, inv) + kRound);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) b[i] = quantize_by_division(element<SDT>(y[i / E].raw, i % E), sc);
    }
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
      w[h] = __byte_perm(__byte_perm(b[4 * h], b[4 * h + 1], 0x0040), __byte_perm(b[4 * h + 2], b[4 * h + 3], 0x0040), 0x5410);
    reinterpret_cast<uint2*>(d)[v] = zero ? make_uint2(0u, 0u) : make_uint2(w[0], w[1]);
  };
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (t + u * G < nvec) store(t + u * G, x[u]);
  for (int v = t + U * G; v < nvec; v += G) {
    Half y[NH];
#pragma unroll
    for (int h = 0; h < NH; ++h) y[h].raw = s[v * NH + h];
    store(v, y);
  }
  if (t < 8 && last < cols) d[last] = zero ? (int8_t)0 : (int8_t)quantize_by_division(tail, sc);
}

template <int SDT>
static cudaError_t launch_quantize(const void* src, int64_t ss, void* dst, int64_t ds, float* scale, int rows, int cols,
                                   cudaStream_t st) {
  // As many warps per row as hold it in four vectors per thread: what a thread does besides its elements (two divisions, the
  // maximum over the warps) costs as much as ten of them.  bf16, 8192 rows of 2048 / 4096: 16.4 / 22.8 us with 256 threads per row.
  auto kern = cols <= 1024 ? quantize_rows_kernel<SDT, 32, 4>
              : cols <= 2048 ? quantize_rows_kernel<SDT, 64, 4>
              : cols <= 4096 ? quantize_rows_kernel<SDT, 128, 4>
              : cols <= 8192 ? quantize_rows_kernel<SDT, 256, 4> : quantize_rows_kernel<SDT, 256, 8>;
  const int per = cols <= 1024 ? 8 : cols <= 2048 ? 4 : cols <= 4096 ? 2 : 1;    // rows per block
  const unsigned blocks = (unsigned)(((int64_t)rows + per - 1) / per);
  return launch_overlapped(kern, dim3(blocks), dim3(256), 0, st, src, ss, (int8_t*)dst, ds, scale, rows, cols);
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
  const int64_t size = dtype_size(src_dtype);
  const RowSpan in{src, rows, cols * size, src_stride * size}, q{dst, rows, cols, dst_stride};
  const RowSpan s{scale, 1, 4 * (int64_t)rows, 4 * (int64_t)rows};
  if (share_memory(in, q) || share_memory(in, s) || share_memory(q, s)) return CFK_ERR_INVALID_ARG;
  const cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e;
  switch (src_dtype) {
    case CFK_FP16: e = launch_quantize<CFK_FP16>(src, src_stride, dst, dst_stride, scale, rows, cols, st); break;
    case CFK_BF16: e = launch_quantize<CFK_BF16>(src, src_stride, dst, dst_stride, scale, rows, cols, st); break;
    default: e = launch_quantize<CFK_FP32>(src, src_stride, dst, dst_stride, scale, rows, cols, st); break;
  }
  return note_cuda(e, "quantize launch") == cudaSuccess ? CFK_OK : CFK_ERR_LAUNCH;
}
