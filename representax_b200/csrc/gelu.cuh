// GELU of the fused epilogues.
#pragma once
#include <cuda_runtime.h>

namespace rx {
namespace gemm {

// GELU (erf form) and its derivative from one exponential: the normal CDF
// Phi(x) = (1 + erf(x / sqrt 2)) / 2 uses the rational approximation of
// Abramowitz & Stegun, Handbook of Mathematical Functions, eq. 7.1.26
// (|error of erf| <= 1.5e-7: an absolute bound, far below bf16's resolution of
// values near one; for x < -4, where Phi is as small as that, the relative error
// is large), whose exp(-u^2) factor at u = |x| / sqrt 2 is exp(-x^2 / 2), the same exponential the normal
// density phi(x) needs. gelu = x Phi(x); gelu' = Phi(x) + x phi(x).
__device__ __forceinline__ void gelu_and_grad(float x, float& gelu, float& grad) {
  const float u = fabsf(x) * 0.70710678118654752440f;
  float t;  // 1 / (1 + p u) by the approximate reciprocal (a few ulp, far below bf16's resolution)
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(0.3275911f, u, 1.0f)));
  float poly = fmaf(1.061405429f, t, -1.453152027f);
  poly = fmaf(poly, t, 1.421413741f);
  poly = fmaf(poly, t, -0.284496736f);
  poly = fmaf(poly, t, 0.254829592f);
  poly *= t;
  float e;  // exp(-x^2 / 2) = 2^(-x^2 / 2 * log2(e))
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-0.72134752044448170368f * x * x));
  const float erf_u = 1.0f - poly * e;  // erf(|x| / sqrt 2)
  const float cdf = 0.5f + 0.5f * copysignf(erf_u, x);
  gelu = x * cdf;
  grad = fmaf(x * 0.39894228040143267794f, e, cdf);
}

}  // namespace gemm
}  // namespace rx
