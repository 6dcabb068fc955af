// Activations in fp32, shared by the operators that round once at the end (linear.hip, ssm.hip).
#pragma once

#include "device_utils.h"

#pragma clang fp contract(off)

namespace frhip {

constexpr float kLog2e = 1.44269504088896340736f;

// exp(-v) for v in [-88, 120], with the rounding of v log2(e), which exp2 would scale by |v|, made good: t + r = v log2(e), log2(e) =
// kLog2e + 1.925963033500752e-8
__device__ __forceinline__ float exp_neg_fine(float v) {
  const float t = v * kLog2e, r = __builtin_fmaf(v, 1.925963033500752e-8f, __builtin_fmaf(v, kLog2e, -t)), e = __builtin_amdgcn_exp2f(-t);
  return __builtin_fmaf(e, r * -0.693147180559945f, e);
}

// log(1 + exp(v)) = max(v, 0) + log1p(e), e = exp(-|v|); log1p(e) = 2 atanh(s), s = e / (2 + e) <= 1/3.  With g = 2 s = e / (1 + e / 2) that is
// g P(g^2), P a polynomial (Chebyshev fit of atanh(s) / s over s^2 in [0, 1/9], 8e-9 relative), so that small values keep their
// relative accuracy.
template <bool FINE>
__device__ __forceinline__ float softplus_f(float v) {
  const float m = __builtin_fabsf(v);
  const float e = FINE ? exp_neg_fine(__builtin_fminf(m, 120.f)) : __builtin_amdgcn_exp2f(m * -kLog2e);  // exp(-120) is no fp32 number
  const float g = e * __builtin_amdgcn_rcpf(__builtin_fmaf(0.5f, e, 1.0f)), q = g * g;
  float p = __builtin_fmaf(q, 0.1408732831478119f / 256, 0.1398070901632309f / 64);
  p = __builtin_fmaf(p, q, 0.20012426376342773f / 16);
  p = __builtin_fmaf(p, q, 0.3333315849304199f / 4);
  p = __builtin_fmaf(p, q, 1.0f);
  const float y = __builtin_fmaf(g, p, __builtin_amdgcn_fmed3f(v, 0.f, __builtin_inff()));  // a NaN stays one through g
  return FINE && v != v ? v : y;
}

// FINE: for results that stay fp32; otherwise within a few units of the instructions for exp2 and the reciprocal, far below what the
// rounding to binary16 takes
template <bool FINE>
__device__ __forceinline__ float sigmoid_f(float v) {
  if constexpr (FINE) {
    const float d = 1.0f + exp_neg_fine(__builtin_fminf(__builtin_fmaxf(v, -88.f), 120.f)), r = __builtin_amdgcn_rcpf(d);
    const float y = __builtin_fmaf(__builtin_fmaf(-d, r, 1.0f), r, r);
    return v == v ? y : v;
  }
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -kLog2e));
}
template <bool FINE>
__device__ __forceinline__ float silu_f(float v) { return v * sigmoid_f<FINE>(v); }

}  // namespace frhip
