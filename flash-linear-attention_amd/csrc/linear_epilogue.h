// What the products of projections do with their sums: activations, values at any address.
#pragma once
#include "fla_common.h"

namespace {

template <int ACT>
FLA_DEVICE float activate(float v) {
  if (ACT == FLA_ACT_SILU) return v * __builtin_amdgcn_rcpf(1.f + __expf(-v));
  if (ACT == FLA_ACT_GELU) return 0.5f * v * (1.f + erff(v * 0.70710678f));
  if (ACT == FLA_ACT_RELU) return v < 0.f ? 0.f : v;      // (NaN stays)
  return v;
}

// erf by Abramowitz and Stegun's formula 7.1.26, |error| <= 1.5e-7 (2^-22.7): a reciprocal, an exponential and seven multiply-adds, where erff takes
// some forty instructions, which an epilogue of 128 values a lane has to wait for.  Returns Phi(v) = (1 + erf(v / sqrt 2)) / 2 and exp(-v^2 / 2).
FLA_DEVICE float normal_cdf(float v, float* bell) {
  const float x = __builtin_fabsf(v) * 0.70710678f, t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, x, 1.f));
  *bell = __expf(-x * x);
  const float tail = 0.5f * t * *bell * fmaf(fmaf(fmaf(fmaf(1.061405429f, t, -1.453152027f), t, 1.421413741f), t, -0.284496736f), t, 0.254829592f);
  return v < 0.f ? tail : 1.f - tail;
}
// the activation of a gate, for results in 16 bits
template <int ACT>
FLA_DEVICE float activate_gate(float v) {
  float bell;
  if (ACT == FLA_ACT_GELU) return v * normal_cdf(v, &bell);
  return activate<ACT>(v);
}
// ... and its derivative
template <int ACT>
FLA_DEVICE float activate_gate(float v, float* slope) {
  if (ACT == FLA_ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.f + __expf(-v));
    *slope = s * fmaf(v, 1.f - s, 1.f);
    return v * s;
  }
  if (ACT == FLA_ACT_GELU) {
    float bell;
    const float c = normal_cdf(v, &bell);
    *slope = fmaf(v * 0.39894228f, bell, c);
    return v * c;
  }
  *slope = ACT == FLA_ACT_RELU && !(v > 0.f) ? (v == v ? 0.f : v) : 1.f;   // (NaN stays)
  return activate<ACT>(v);
}

// COUNT values at any element address; unless FULL, the first `valid` of them one by one
template <typename T, int COUNT, bool FULL>
FLA_DEVICE void load_some(const T* p, int valid, float* o) {
  if (FULL) {
    typedef T vec __attribute__((ext_vector_type(COUNT), aligned(alignof(T))));
    const vec v = *(const vec*)p;
#pragma unroll
    for (int i = 0; i < COUNT; ++i) o[i] = (float)v[i];
  } else {
#pragma unroll
    for (int i = 0; i < COUNT; ++i) o[i] = i < valid ? (float)p[i] : 0.f;
  }
}

// the activation as a constant: one branch a tile instead of one an element
template <int V>
struct Const {
  static constexpr int value = V;
};
template <typename F>
FLA_DEVICE void with_activation(int act, const F& f) {
  if (act == FLA_ACT_SILU) f(Const<FLA_ACT_SILU>());
  else if (act == FLA_ACT_GELU) f(Const<FLA_ACT_GELU>());
  else if (act == FLA_ACT_RELU) f(Const<FLA_ACT_RELU>());
  else f(Const<FLA_ACT_NONE>());
}

// the same where a kernel is made for one activation (ACT; -1: for all)
template <int ACT, typename F>
FLA_DEVICE void with_this_activation(int act, const F& f) {
  if constexpr (ACT >= 0) f(Const<ACT>());
  else with_activation(act, f);
}
// f(Const<activation>), on the host
template <typename F>
int for_activation(int act, const F& f) {
  return act == FLA_ACT_SILU ? f(Const<FLA_ACT_SILU>()) : act == FLA_ACT_GELU ? f(Const<FLA_ACT_GELU>()) : act == FLA_ACT_RELU ? f(Const<FLA_ACT_RELU>())
                                                                                                        : f(Const<FLA_ACT_NONE>());
}

}  // namespace
