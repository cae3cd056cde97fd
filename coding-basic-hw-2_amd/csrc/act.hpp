// act.hpp -- activations of gated feed-forward blocks and their slopes, in 32 bits.
#pragma once
#include "common.hpp"
#include "ggemm_glu.h"

namespace ggemm {

inline bool act_known(int act) { return act == GGEMM_SILU || act == GGEMM_GELU || act == GGEMM_GELU_TANH; }

// f(integral_constant<int, ACT>) for the activation of a call
template <class F>
inline void with_act(int act, F&& f) {
  if (act == GGEMM_SILU) f(std::integral_constant<int, GGEMM_SILU>{});
  else if (act == GGEMM_GELU) f(std::integral_constant<int, GGEMM_GELU>{});
  else f(std::integral_constant<int, GGEMM_GELU_TANH>{});
}

// 1 / (1 + exp(-z)).  exp2 and the reciprocal are the hardware's (1 ulp each); the argument's rounding adds
// |z| 2^-24 relative.  exp(-z) = Inf gives 0.
__device__ __forceinline__ float logistic(float z) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * z));
}

// act(v) = v p(v); act'(v) = p(v) + v p'(v).  Gives p and p'.
//   SILU       p = logistic(v),             p' = p (1 - p)
//   GELU       p = Phi(v), the normal distribution's, p' = its density.  By Abramowitz and Stegun 7.1.26: with
//              x = |v| / sqrt 2, t = 1 / (1 + 0.3275911 x): erfc(x) = (a1 t + .. + a5 t^5) exp(-x^2), off by at most
//              1.5e-7; p = 1 - erfc / 2 or erfc / 2 by v's sign.  Nine multiply-adds and the density's exponential, where
//              a library error function takes several times that in the epilogue of every tile.  v p is off by 4.2e-7 at most
//              (at 3.06; of itself, 3e-6 above -2, 5e-5 above -3, 2e-3 above -5, 1e-2 above -8).
//   GELU_TANH  p = logistic(2 z), z = sqrt(2 / pi) (v + 0.044715 v^3), p' = p (1 - p) 2 z'.  Past |v| = 16, p is 0 or 1 to the
//              last bit; the clamp keeps v^3 and z' finite, so that no 0 Inf arises.
template <int ACT>
__device__ __forceinline__ void act_parts(float v, float& p, float& dp) {
  if constexpr (ACT == GGEMM_SILU) {
    p = logistic(v);
    dp = p * (1.0f - p);
  } else if constexpr (ACT == GGEMM_GELU) {
    const float x = fabsf(v) * 0.70710678f, e = __builtin_amdgcn_exp2f(-0.72134752f * v * v);
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, x, 1.0f));
    const float s = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
    const float half = 0.5f * s * e;
    p = v < 0.0f ? half : 1.0f - half;
    dp = 0.39894228f * e;
  } else {
    const float c = fminf(fmaxf(v, -16.0f), 16.0f), w = c * c;
    p = logistic(1.59576912f * c * fmaf(0.044715f, w, 1.0f));
    dp = p * (1.0f - p) * 1.59576912f * fmaf(0.134145f, w, 1.0f);
  }
}
template <int ACT>
__device__ __forceinline__ float act_value(float v) {
  float p, dp;
  act_parts<ACT>(v, p, dp);
  return v * p;
}

}  // namespace ggemm
