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

// Phi(v) = (1 + erf(v / sqrt 2)) / 2 and exp(-v^2 / 2).  The tail Phi(-|v|) is that bell times t P(t), t = 1 / (1 + 0.3058 |v|) (the form of Abramowitz and Stegun's
// formula 7.1.26, whose five coefficients hold an absolute error of 1.5e-7 alone: 1.6e-3 of the tail at -5).  P: the minimax fit of the relative error
// over |v| <= 14.8, a linear program over 6000 points, 7.9e-8.  With the roundings of v^2 in the exponent the tail is within (1.25 v^2 + 16) 2^-24 of itself.  A
// reciprocal, an exponential and nine multiply-adds, where erff takes some forty instructions, which an epilogue of 128 values a lane has to wait for.
FLA_DEVICE float normal_cdf(float v, float* bell) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.3058f, __builtin_fabsf(v), 1.f));
  *bell = __builtin_amdgcn_exp2f(v * v * -0.72134752f);
  float p = fmaf(0.0366655402f, t, -0.151510358f);
  p = fmaf(p, t, 0.181176946f), p = fmaf(p, t, -0.0344329774f), p = fmaf(p, t, 0.119286954f);
  p = fmaf(p, t, 0.104134202f), p = fmaf(p, t, 0.122716859f), p = fmaf(p, t, 0.121962912f);
  const float tail = t * p * *bell;
  return v < 0.f ? tail : 1.f - tail;
}
// the activation of a gate and of products of integers, for results in 16 and in 32 bits
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
