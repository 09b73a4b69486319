// The activations of the gated feed-forward block and their derivatives, in fp32.
//   SiLU x s(x), GELU_TANH x s(2a(x)) with a = sqrt(2/pi) (x + 0.044715 x^3), since (1 + tanh a) / 2 = s(2a), s the logistic
//   function; GELU x Phi(x) with Phi(x) = erfc(-x / sqrt 2) / 2, which keeps its relative accuracy where 1 + erf would cancel.
// s is computed as 1 / (1 + 2^(-x log2 e)) with the special-function unit: relative error below 1e-6 for |x| < 10, growing with |x| to 1e-5
// where s is about to underflow; an exponential that overflows gives s = 0, as it should.
#pragma once
#include "common.cuh"
#include "../../include/cfk_b200.h"

namespace cfk {

__device__ __forceinline__ float logistic(float x) { return __fdividef(1.f, 1.f + ex2_approx(-1.4426950408889634f * x)); }
__device__ __forceinline__ float gelu_tanh_2a(float x) { return x * (1.5957691216057308f + 0.0713548162726f * x * x); }

template <int ACT>
__device__ __forceinline__ float activate(float x) {
  if constexpr (ACT == CFK_ACT_SILU) return x * logistic(x);
  else if constexpr (ACT == CFK_ACT_GELU_TANH) return x * logistic(gelu_tanh_2a(x));
  else if constexpr (ACT == CFK_ACT_GELU) return 0.5f * x * erfcf(-0.70710678118654752f * x);
  else return x < 0.f ? 0.f : x;                 // NaN stays
}

// value and derivative
template <int ACT>
__device__ __forceinline__ float2 activate_grad(float x) {
  if constexpr (ACT == CFK_ACT_SILU) {
    const float s = logistic(x), v = x * s;
    const float tail = s * (1.f - s);
    return make_float2(v, s + (tail == 0.f ? 0.f : x * tail));
  } else if constexpr (ACT == CFK_ACT_GELU_TANH) {
    const float s = logistic(gelu_tanh_2a(x)), tail = s * (1.f - s);
    // where s has reached 0 or 1 the slope of its argument no longer counts (and may have overflowed)
    const float bend = tail == 0.f ? 0.f : x * tail * (1.5957691216057308f + 0.2140644488178f * x * x);
    return make_float2(x * s, s + bend);
  } else if constexpr (ACT == CFK_ACT_GELU) {
    const float cdf = 0.5f * erfcf(-0.70710678118654752f * x);
    const float pdf = 0.3989422804014327f * ex2_approx(-0.72134752044448170f * x * x);
    return make_float2(x * cdf, cdf + (pdf == 0.f ? 0.f : x * pdf));
  } else {
    return make_float2(x < 0.f ? 0.f : x, x > 0.f ? 1.f : (x <= 0.f ? 0.f : x));
  }
}

}  // namespace cfk
