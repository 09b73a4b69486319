// Elementwise arithmetic of the feed-forward products: scales of integer sums, activations and their derivatives, in fp32.
//
//   SiLU x s(x), GELU_TANH x s(2a(x)) with a = sqrt(2/pi) (x + 0.044715 x^3), since (1 + tanh a) / 2 = s(2a), s the logistic
//   function; GELU x Phi(x) with Phi(x) = erfc(-x / sqrt 2) / 2, which keeps its relative accuracy where 1 + erf would cancel.
// With r = 2^(-|x| log2(e) / 2): s(|x|) = 1 / (1 + r^2), s(-|x|) = r^2 / (1 + r^2), by the special-function unit, whose divisor stays in
// [1, 2].  e^-|x| itself is never held: a product with it takes the two factors r one after the other, so x s(x) and the
// derivatives underflow where they themselves leave the range of fp32 and not where s does, a large factor behind them
// finds their value (gate -90 beside up 1e37), and an r that is 0 gives 0.  Relative error below 1e-6 for |x| < 10, growing with the
// exponent to 2e-5 where r underflows (7e-5 in the tanh form, whose exponent is a polynomial); for GELU, whose erfc is subnormal from
// x = -13 on, 2e-5 or 2^-145 absolute.
#pragma once
#include "common.cuh"
#include "../../include/cfk_b200.h"

namespace cfk {

// A row's scale, which multiplies an integer sum ahead of the column's: scale = by * rest.  Beside a scale of 2^64 or more a sum could
// pass the range of fp32 although its product with a small column scale does not, so 2^32 of it are left for the end.  (Below, a
// sum of up to 2^31 stays under 2^95; a sum times a subnormal scale is exact or normal, so nothing is lost at the other end.)
struct RowScale { float by, rest; };
__device__ __forceinline__ RowScale split_row_scale(float s) {
  const bool large = fabsf(s) >= 18446744073709551616.f;
  return RowScale{large ? s * 2.3283064365386963e-10f : s, large ? 4294967296.f : 1.f};
}

// s(z) = d a^2
struct Logistic { float r, d, a; };
__device__ __forceinline__ Logistic logistic(float z) {
  Logistic l;
  l.r = ex2_approx(-0.72134752044448170f * fabsf(z));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(l.d) : "f"(fmaf(l.r, l.r, 1.f)));
  l.a = z < 0.f ? l.r : 1.f;
  return l;
}
__device__ __forceinline__ float gelu_tanh_2a(float x) { return x * (1.5957691216057308f + 0.0713548162726f * x * x); }
// v = x s(z), and with z' of z(x) its derivative s + x z' s (1 - s) = s (1 + z' (x - v)).  s has reached 1, and x - v is 0, where z passes
// 17: until there the rounding of v costs 2e-6 of the slope at most.  Where r is 0 the second term no longer counts (x or z' may be
// infinite).
__device__ __forceinline__ float logistic_times(float x, const Logistic& l) { return x * (l.d * l.a) * l.a; }
__device__ __forceinline__ float2 logistic_grad(float x, float slope, const Logistic& l) {
  const float v = logistic_times(x, l), bend = l.r == 0.f ? 0.f : slope * (x - v);
  return make_float2(v, (1.f + bend) * (l.d * l.a) * l.a);
}

template <int ACT>
__device__ __forceinline__ float activate(float x) {
  if constexpr (ACT == CFK_ACT_SILU) return logistic_times(x, logistic(x));
  else if constexpr (ACT == CFK_ACT_GELU_TANH) return logistic_times(x, logistic(gelu_tanh_2a(x)));
  else if constexpr (ACT == CFK_ACT_GELU) return 0.5f * x * erfcf(-0.70710678118654752f * x);
  else return x < 0.f ? 0.f : x;                 // NaN stays
}

// value and derivative
template <int ACT>
__device__ __forceinline__ float2 activate_grad(float x) {
  if constexpr (ACT == CFK_ACT_SILU) {
    return logistic_grad(x, 1.f, logistic(x));
  } else if constexpr (ACT == CFK_ACT_GELU_TANH) {
    return logistic_grad(x, 1.5957691216057308f + 0.2140644488178f * x * x, logistic(gelu_tanh_2a(x)));
  } else if constexpr (ACT == CFK_ACT_GELU) {
    const float cdf = 0.5f * erfcf(-0.70710678118654752f * x);
    const float r = ex2_approx(-0.36067376022224085f * x * x);           // the density is 0.399 r^2
    return make_float2(x * cdf, cdf + (r == 0.f ? 0.f : 0.3989422804014327f * x * r * r));
  } else {
    return make_float2(x < 0.f ? 0.f : x, x > 0.f ? 1.f : (x <= 0.f ? 0.f : x));
  }
}

}  // namespace cfk
