// Activations of the gated feed-forward kernels: the value act(g) and the
// derivative act'(g) in fp32 from one exponential.
//
//   silu        g s(g),          s(x) = 1 / (1 + exp(-x))
//   quick gelu  g s(1.702 g)
//   gelu (tanh) g s(2 v), v = sqrt(2 / pi) (g + 0.044715 g^3), since (1 + tanh v) / 2 = s(2 v)
//   gelu (erf)  g Phi(g)
//
// The codes are those of the elementwise kernels (pointwise.cu). The results
// are held in at most 16 bits afterwards, each relative to its own magnitude or
// to that of a block of 32, so what is asked of the fast exponential and
// reciprocal is a small relative error, in the negative tails too: below 2e-5
// (2^-15.6) while the exponential is a normal number (g > -13 for the erf form).
#pragma once
#include <cuda_runtime.h>

namespace rx {
namespace gated {

enum Act : int { kGeluErf = 0, kGeluTanh = 1, kSilu = 2, kQuickGelu = 3 };

template <int ACT>
struct ActCode {
  static constexpr int value = ACT;
};

__device__ __forceinline__ float logistic(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }

// Phi(g) and exp(-g^2 / 2). The lower tail is Phi(-u) = exp(-u^2 / 2) t P(t), t = 1 / (1 + 0.38 u): P is the
// degree-6 polynomial whose relative error over u in [0, 40] is the smallest (minimax fit by linear programming in
// 64 bits: 2.5e-6). It is taken as it is for g < 0, where 1 - (...) would leave nothing of it.
__device__ __forceinline__ float normal_cdf(float g, float& e) {
  float t;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(0.38f, fabsf(g), 1.f)));
  float poly = fmaf(0.0489545763f, t, -0.1600402f);
  poly = fmaf(poly, t, 0.114407621f);
  poly = fmaf(poly, t, 0.0599808581f);
  poly = fmaf(poly, t, 0.133793741f);
  poly = fmaf(poly, t, 0.151299015f);
  poly = fmaf(poly, t, 0.151605666f);
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-0.72134752044448170368f * g * g));  // -log2(e) / 2
  const float tail = poly * t * e;
  return g < 0.f ? tail : 1.f - tail;
}

template <int ACT>
__device__ __forceinline__ float act_value(float g) {
  if constexpr (ACT == kGeluErf) {
    float e;
    return g * normal_cdf(g, e);
  }
  if constexpr (ACT == kGeluTanh) return g * logistic(1.5957691216057308f * fmaf(0.044715f * g * g, g, g));
  if constexpr (ACT == kSilu) return g * logistic(g);
  return g * logistic(1.702f * g);
}

template <int ACT>
__device__ __forceinline__ void act_value_grad(float g, float& value, float& grad) {
  if constexpr (ACT == kGeluErf) {
    float e;
    const float cdf = normal_cdf(g, e);
    value = g * cdf;
    grad = fmaf(g * 0.39894228040143267794f, e, cdf);  // Phi + g phi
  } else if constexpr (ACT == kGeluTanh) {
    const float s = logistic(1.5957691216057308f * fmaf(0.044715f * g * g, g, g));
    value = g * s;
    grad = fmaf(g * s * (1.f - s), 1.5957691216057308f * fmaf(0.134145f * g, g, 1.f), s);
  } else {
    constexpr float k = ACT == kSilu ? 1.f : 1.702f;
    const float s = logistic(k * g);
    value = g * s;
    grad = fmaf(k * g * s, 1.f - s, s);
  }
}

// f(integral_constant of the activation): the choice is made once for a run of values, not for each.
template <typename F>
__device__ __forceinline__ void with_act(int act, F&& f) {
  switch (act) {
    case kGeluErf: f(ActCode<kGeluErf>{}); return;
    case kGeluTanh: f(ActCode<kGeluTanh>{}); return;
    case kSilu: f(ActCode<kSilu>{}); return;
    default: f(ActCode<kQuickGelu>{}); return;
  }
}

// v[i] = act(g[i]) * v[i]
template <int N>
__device__ __forceinline__ void gate(int act, const float (&g)[N], float (&v)[N]) {
  with_act(act, [&](auto code) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] *= act_value<decltype(code)::value>(g[i]);
  });
}

// a = act(g), b = act'(g) * u, u becomes act(g) * u (g holds a afterwards)
template <int N>
__device__ __forceinline__ void gate_and_keep(int act, float (&g)[N], float (&u)[N], float (&b)[N]) {
  with_act(act, [&](auto code) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float value, grad;
      act_value_grad<decltype(code)::value>(g[i], value, grad);
      g[i] = value;
      b[i] = u[i] * grad;
      u[i] *= value;
    }
  });
}

}  // namespace gated
}  // namespace rx
