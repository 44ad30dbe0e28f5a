// Eight consecutive elements of a row in a lane's registers, and sums over the lanes that hold a row.
#pragma once
#include "fla_common.h"

namespace {

constexpr int VEC = 8;

template <typename T>
struct Row8;
template <>
struct Row8<float> {
  struct raw {
    f32x4 a, b;
  };
  static FLA_DEVICE raw load_raw(const float* p) { return raw{*(const f32x4*)p, *(const f32x4*)(p + 4)}; }
  static FLA_DEVICE void unpack(const raw& r, float* o) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[i] = r.a[i];
      o[4 + i] = r.b[i];
    }
  }
  static FLA_DEVICE void load(const float* p, float* o) {
    f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[i] = a[i];
      o[4 + i] = b[i];
    }
  }
  static FLA_DEVICE void store(float* p, const float* v) {
    *(f32x4*)p = f32x4{v[0], v[1], v[2], v[3]};
    *(f32x4*)(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
  }
};
template <>
struct Row8<bf16> {
  typedef bf16x8 raw;
  static FLA_DEVICE raw load_raw(const bf16* p) { return *(const bf16x8*)p; }
  static FLA_DEVICE void unpack(const raw& r, float* o) {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (float)r[i];
  }
  static FLA_DEVICE void load(const bf16* p, float* o) {
    bf16x8 a = *(const bf16x8*)p;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (float)a[i];
  }
  static FLA_DEVICE void store(bf16* p, const float* v) {
    bf16x8 a;
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = (bf16)v[i];
    *(bf16x8*)p = a;
  }
};
template <>
struct Row8<f16> {
  typedef f16x8 raw;
  static FLA_DEVICE raw load_raw(const f16* p) { return *(const f16x8*)p; }
  static FLA_DEVICE void unpack(const raw& r, float* o) {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (float)r[i];
  }
  static FLA_DEVICE void load(const f16* p, float* o) {
    f16x8 a = *(const f16x8*)p;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (float)a[i];
  }
  static FLA_DEVICE void store(f16* p, const float* v) {
    f16x8 a;
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = (f16)v[i];
    *(f16x8*)p = a;
  }
};

// Eight elements at p of which the first `valid` exist, the others as `fill` (<= 0: none, p is not read).  WIDE: p is aligned to 16 bytes
// and valid is 8 or more, or not positive; otherwise any element address goes, whole pieces in one load all the same.
template <typename T, bool WIDE>
FLA_DEVICE typename Row8<T>::raw load_raw8(const T* p, int valid, float fill = 0.f) {
  typename Row8<T>::raw r;
  if (WIDE && valid > 0) return Row8<T>::load_raw(p);
  if (!WIDE && valid >= VEC) {
    typedef T any8 __attribute__((ext_vector_type(8), aligned(alignof(T))));
    const any8 v = *(const any8*)p;
    __builtin_memcpy(&r, &v, sizeof r);
    return r;
  }
  T e[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) e[i] = !WIDE && i < valid ? p[i] : (T)fill;
  __builtin_memcpy(&r, e, sizeof r);
  return r;
}
template <typename T, bool WIDE>
FLA_DEVICE void store8(T* p, const float* v, int valid) {
  if (WIDE) {
    if (valid > 0) Row8<T>::store(p, v);
  } else if (valid >= VEC) {
    typedef T any8 __attribute__((ext_vector_type(8), aligned(alignof(T))));
    any8 o;
#pragma unroll
    for (int i = 0; i < VEC; ++i) o[i] = (T)v[i];
    *(any8*)p = o;
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (i < valid) p[i] = (T)v[i];
  }
}

// sum over the LPR lanes of a group (LPR a power of two <= 64), result in every lane
template <int LPR>
FLA_DEVICE float group_sum(float x) {
#pragma unroll
  for (int m = LPR / 2; m >= 1; m >>= 1) x += __shfl_xor(x, m, 64);
  return x;
}

// the hardware reciprocal (1 ulp) instead of an IEEE division: ten instructions less per element
FLA_DEVICE float sigmoidf(float x) { return __builtin_amdgcn_rcpf(1.f + __expf(-x)); }

}  // namespace
