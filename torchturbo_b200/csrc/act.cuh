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
// packed form, and erf by Abramowitz and Stegun 7.1.26 (C. Hastings),
//   erfc(x) = (a1 t + ... + a5 t^5) exp(-x^2) + e,  t = 1 / (1 + p x),  x >= 0,  |e| <= 1.5e-7,
// a fortieth of the smallest step of bf16 next to 1, whose exponential the derivative of gelu takes as well.
struct GeluErf {
  float upper, expo;     // 1 - Phi(|v|), exp(-v^2 / 2)
};
__device__ __forceinline__ GeluErf gelu_erf_parts(float v) {
  const float a = fabsf(v);
  const float t = __fdividef(1.f, fmaf(a, 0.3275911f * 0.7071067811865476f, 1.f));
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v * v * (-0.5f * 1.4426950408889634f)));
  float q = fmaf(t, 0.5f * 1.061405429f, -0.5f * 1.453152027f);
  q = fmaf(q, t, 0.5f * 1.421413741f);
  q = fmaf(q, t, -0.5f * 0.284496736f);
  q = fmaf(q, t, 0.5f * 0.254829592f);
  return GeluErf{q * t * e, e};
}
__device__ __forceinline__ float tanh_approx(float x) {
  float y;
  asm("tanh.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// (a, b) -> act(a), act(b)
template <int ACT>
__device__ __forceinline__ void act_pair(float& a, float& b) {
  if (ACT == 1) {
    // 0.5 v (1 + tanh(v (c + 0.044715 c v^2)))
    const uint64_t v = f2_pack(a, b), h = f2_mul(v, f2_pack(0.5f, 0.5f));
    float ua, ub;
    f2_unpack(f2_mul(v, f2_fma(f2_mul(v, v), f2_pack(0.035677408136300125f, 0.035677408136300125f), f2_pack(0.7978845608028654f, 0.7978845608028654f))), ua, ub);
    f2_unpack(f2_fma(h, f2_pack(tanh_approx(ua), tanh_approx(ub)), h), a, b);
  } else if (ACT == 2) {
    const float qa = gelu_erf_parts(a).upper, qb = gelu_erf_parts(b).upper;
    a *= a > 0.f ? 1.f - qa : qa;
    b *= b > 0.f ? 1.f - qb : qb;
  }
}
template <int ACT>
__device__ __forceinline__ float act_slope(float v) {
  if (ACT == 1) {
    // with u = v (c + k v^2), t = tanh u:  0.5 (1 + t) + 0.5 v (1 - t^2) (c + 3 k v^2)
    const float v2 = v * v, t = tanh_approx(v * fmaf(v2, 0.035677408136300125f, 0.7978845608028654f));
    return fmaf(fmaf(-t, t, 1.f) * v, fmaf(v2, 1.5f * 0.035677408136300125f, 0.5f * 0.7978845608028654f), fmaf(t, 0.5f, 0.5f));
  }
  if (ACT == 2) {
    const GeluErf g = gelu_erf_parts(v);
    return fmaf(v * 0.3989422804014327f, g.expo, v > 0.f ? 1.f - g.upper : g.upper);
  }
  return 1.f;
}

}  // namespace ttb
