// Activations of the gated feed-forward kernels: the value act(g) and the
// derivative act'(g) in fp32 from one exponential.
//
//   silu        g s(g),          s(x) = 1 / (1 + exp(-x))
//   quick gelu  g s(1.702 g)
//   gelu (tanh) g s(2 v), v = sqrt(2 / pi) (g + 0.044715 g^3), since (1 + tanh v) / 2 = s(2 v)
//   gelu (erf)  g Phi(g), see gelu_and_grad in gelu.cuh
//
// The codes are those of the elementwise kernels (pointwise.cu). The results
// are held in at most 16 bits afterwards, so the fast exponential and
// reciprocal (a few ulp of fp32) lose nothing.
#pragma once
#include "gelu.cuh"

namespace rx {
namespace gated {

enum Act : int { kGeluErf = 0, kGeluTanh = 1, kSilu = 2, kQuickGelu = 3 };

__device__ __forceinline__ float logistic(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }

__device__ __forceinline__ float act_value(float g, int act) {
  switch (act) {
    case kGeluErf: return gemm::gelu_erf(g);
    case kGeluTanh: return g * logistic(1.5957691216057308f * fmaf(0.044715f * g * g, g, g));
    case kSilu: return g * logistic(g);
    default: return g * logistic(1.702f * g);
  }
}

__device__ __forceinline__ void act_value_grad(float g, int act, float& value, float& grad) {
  switch (act) {
    case kGeluErf: gemm::gelu_and_grad(g, value, grad); return;
    case kGeluTanh: {
      const float s = logistic(1.5957691216057308f * fmaf(0.044715f * g * g, g, g));
      value = g * s;
      grad = fmaf(g * s * (1.f - s), 1.5957691216057308f * fmaf(0.134145f * g, g, 1.f), s);
      return;
    }
    case kSilu: {
      const float s = logistic(g);
      value = g * s;
      grad = fmaf(g * s, 1.f - s, s);
      return;
    }
    default: {
      const float s = logistic(1.702f * g);
      value = g * s;
      grad = fmaf(1.702f * g * s, 1.f - s, s);
      return;
    }
  }
}

}  // namespace gated
}  // namespace rx
