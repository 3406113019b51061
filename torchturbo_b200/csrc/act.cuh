// Activations of biased projections.  0: identity, 1: GELU (tanh approximation), 2: GELU (erf)
#pragma once
#include "common.cuh"

namespace ttb {

__device__ __forceinline__ float act_fwd(float v, int act) {
  if (act == 1) {
    const float u = 0.7978845608028654f * (v + 0.044715f * v * v * v);
    return 0.5f * v * (1.f + tanhf(u));
  }
  if (act == 2) return 0.5f * v * (1.f + erff(v * 0.7071067811865476f));
  return v;
}
__device__ __forceinline__ float act_grad(float v, int act) {
  if (act == 1) {
    const float u = 0.7978845608028654f * (v + 0.044715f * v * v * v);
    const float t = tanhf(u);
    return 0.5f * (1.f + t) + 0.5f * v * (1.f - t * t) * 0.7978845608028654f * (1.f + 3.f * 0.044715f * v * v);
  }
  if (act == 2) return 0.5f * (1.f + erff(v * 0.7071067811865476f)) + v * 0.3989422804014327f * __expf(-0.5f * v * v);
  return 1.f;
}

// The same for pairs of values in the epilogue of a product and in its backward, where the arithmetic is the bound: half of the products in
// packed form.
//   tanh  (1 + tanh u) / 2 = 1 / (1 + exp(-2 u)), which does not cancel where u is far below zero: values and slopes keep 2^-17 and 2^-15 of
//         their own size from -6 on.  The hardware's hyperbolic tangent (one instruction for two) is 2^-11 off, more than all of the value at -4.
//   erf   by Abramowitz and Stegun 7.1.26 (C. Hastings),  erfc(x) = (a1 t + ... + a5 t^5) exp(-x^2) + e,  t = 1 / (1 + p x),  x >= 0,
//         |e| <= 1.5e-7: relative to gelu's value 0.03 of half a step of bf16 (2^-9 next to 1) at -3, 0.25 at -4, 0.8 at -5 and 2 at -6, where the
//         value is 6e-9.  The derivative takes the same exponential.
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint64_t f2_both(float a) { return f2_pack(a, a); }

// 1 - Phi(|v|) and exp(-v^2 / 2) of two values
__device__ __forceinline__ void gelu_erf_parts(float va, float vb, uint64_t& upper, uint64_t& expo) {
  const uint64_t v = f2_pack(va, vb);
  float a, b;
  f2_unpack(f2_fma(f2_pack(fabsf(va), fabsf(vb)), f2_both(0.3275911f * 0.7071067811865476f), f2_both(1.f)), a, b);
  const uint64_t t = f2_pack(rcp_approx(a), rcp_approx(b));
  f2_unpack(f2_mul(f2_mul(v, v), f2_both(-0.5f * 1.4426950408889634f)), a, b);
  expo = f2_pack(exp2_approx(a), exp2_approx(b));
  uint64_t q = f2_fma(t, f2_both(0.5f * 1.061405429f), f2_both(-0.5f * 1.453152027f));
  q = f2_fma(q, t, f2_both(0.5f * 1.421413741f));
  q = f2_fma(q, t, f2_both(-0.5f * 0.284496736f));
  q = f2_fma(q, t, f2_both(0.5f * 0.254829592f));
  upper = f2_mul(f2_mul(q, t), expo);
}
// s = (1 + tanh u) / 2,  u = v (c + 0.044715 c v^2),  of two values
__device__ __forceinline__ uint64_t gelu_tanh_share(uint64_t v) {
  const float down = -2.f * 1.4426950408889634f;
  float a, b;
  f2_unpack(f2_mul(v, f2_fma(f2_mul(v, v), f2_both(down * 0.035677408136300125f), f2_both(down * 0.7978845608028654f))), a, b);
  f2_unpack(f2_add(f2_pack(exp2_approx(a), exp2_approx(b)), f2_both(1.f)), a, b);
  return f2_pack(rcp_approx(a), rcp_approx(b));
}
// (a, b) -> act(a), act(b)
template <int ACT>
__device__ __forceinline__ void act_pair(float& a, float& b) {
  if (ACT == 1) {
    // v s; of minus infinity none is left
    f2_unpack(f2_mul(f2_pack(fmaxf(a, -3e38f), fmaxf(b, -3e38f)), gelu_tanh_share(f2_pack(a, b))), a, b);
  } else if (ACT == 2) {
    // v Phi(v) = max(v, 0) - |v| (1 - Phi(|v|)); the second term of infinity is none
    uint64_t upper, expo;
    gelu_erf_parts(a, b, upper, expo);
    const float big = 3e38f;
    f2_unpack(f2_fma(f2_pack(-fabsf(fminf(a, big)), -fabsf(fminf(b, big))), upper, f2_pack(fmaxf(a, 0.f), fmaxf(b, 0.f))), a, b);
  }
}
// (a, b) -> act'(a), act'(b)
template <int ACT>
__device__ __forceinline__ void act_slope_pair(float& a, float& b) {
  const uint64_t v = f2_pack(a, b);
  if (ACT == 1) {
    // s + s (1 - s) v 2 u',  2 u' = 2 c + 6 k v^2; from 16 on the second term is below 1e-100, so v^3 stops there
    const uint64_t s = gelu_tanh_share(v);
    const float most = 16.f;
    const uint64_t w = f2_pack(fmaxf(fminf(a, most), -most), fmaxf(fminf(b, most), -most));
    const uint64_t inner = f2_mul(w, f2_fma(f2_mul(w, w), f2_both(6.f * 0.035677408136300125f), f2_both(2.f * 0.7978845608028654f)));
    f2_unpack(f2_fma(f2_fma(f2_mul(s, f2_both(-1.f)), s, s), inner, s), a, b);
  } else if (ACT == 2) {
    // Phi(v) + v phi(v),  Phi(v) = v > 0 ? 1 - upper : upper
    uint64_t upper, expo;
    gelu_erf_parts(a, b, upper, expo);
    float qa, qb;
    f2_unpack(upper, qa, qb);
    f2_unpack(f2_fma(f2_mul(v, f2_both(0.3989422804014327f)), expo, f2_pack(a > 0.f ? 1.f - qa : qa, b > 0.f ? 1.f - qb : qb)), a, b);
  }
}

}  // namespace ttb
