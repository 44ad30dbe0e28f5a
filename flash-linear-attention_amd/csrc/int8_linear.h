// Product of rows in 8-bit integers with the epilogue of a projection:
//   y[m,n] = act(sx[m] sw[n] sum_k x[m,k] w[n,k] + bias[n]) + residual[m,n],   a scale per row of x (token) and of w (channel), act: none, silu, gelu, relu
// Sums are exact in 32 bits: K is at most 131056, where 128 * 128 * K is still below 2^31.  They are rounded to fp32 once (2^-24), and scaled, activated and
// added to the residual there; results leave in 16 bits or in fp32.  8191 x 2048 x 5632: 90 - 98 us, 1.9 - 2.1 POP/s (torch's int8 product of 8192^3: 2.1).  48 x 2048 x 8192 with bias
// and residual 8.8 us (w in the last-level cache), 1 x 4096 x 2048 4.  The tiles of matrix_tiles.h and, up to 64 rows of x, the panels of matrix_panels.h.
#pragma once
#include "linear_epilogue.h"
#include "matrix_panels.h"
#include "matrix_plan.h"
#include "matrix_tiles.h"

namespace {

struct Int8Params {
  const char *x, *w;
  const float *sx, *sw;
  const void *bias, *res;   // or NULL
  void* y;
  int* part;                // [splits, M, N]: sums of a slice of K, or NULL
  int64_t M, N, K;
  int bias_f32, res_f32, act, splits;
  bool res_wide;            // rows of the residual in whole pieces of four elements
};

// Four consecutive n of the residual's row m.  Rows and columns that do not exist are taken from those next to them and not used: no branches.
template <typename R>
FLA_DEVICE f32x4 residual4(const Int8Params& p, int64_t m, int64_t n) {
  const R* row = (const R*)p.res + (m < p.M ? m : p.M - 1) * p.N;
  if (p.res_wide) {
    typedef R V4 __attribute__((ext_vector_type(4)));
    const V4 v = *(const V4*)(row + (n < p.N ? n : p.N - 4));
    return f32x4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
  }
  f32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = (float)row[n + i < p.N ? n + i : p.N - 1];
  return r;
}
template <typename O>
FLA_DEVICE f32x4 int8_residual(const Int8Params& p, int64_t m, int64_t n) {
  if (!p.res) return f32x4{0.f, 0.f, 0.f, 0.f};
  return p.res_f32 ? residual4<float>(p, m, n) : residual4<O>(p, m, n);
}
// Four consecutive n of a row from their sums
template <int ACT>
FLA_DEVICE void int8_values(i32x4 sums, float sx, f32x4 sw, f32x4 bias, f32x4 res, float* v) {
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const float t = fmaf((float)sums[r], sx * sw[r], bias[r]);
    v[r] = activate_gate<ACT>(t) + res[r];
  }
}
template <typename O>
FLA_DEVICE void int8_store4(const Int8Params& p, int64_t m, int64_t n, const float* v) {
  if (m >= p.M) return;
  O* y = (O*)p.y + m * p.N + n;
  if (n + 4 <= p.N) {
    typedef O V4 __attribute__((ext_vector_type(4), aligned(alignof(O))));
    *(V4*)y = V4{(O)v[0], (O)v[1], (O)v[2], (O)v[3]};
  } else {
    f32x4 t = {v[0], v[1], v[2], v[3]};
    const int count = (int)(p.N - n);
#pragma unroll 1
    for (int r = 0; r < count; ++r) {
      y[r] = (O)t[0];
      t[0] = t[1], t[1] = t[2], t[2] = t[3];
    }
  }
}
template <typename O>
FLA_DEVICE float int8_bias(const Int8Params& p, int64_t n) {
  return !p.bias || n >= p.N ? 0.f : p.bias_f32 ? ((const float*)p.bias)[n] : (float)((const O*)p.bias)[n];
}

// RES: a residual is added; ACT: the activation, or -1 for any
template <typename O, int BM, int BN, bool HALVES, bool RES, int ACT>
struct Int8Job {
  static constexpr bool kHalves = HALVES;
  typedef MatTile<int8_t, BM, BN, 2, false, false> Whole;
  typedef MatTile<int8_t, BM, HALVES ? BN / 2 : BN, 2, false, false> Half;
  static constexpr int LATER = Whole::MT * Whole::NT * 2;   // stores of 16-bit results
  static constexpr int kLds = Whole::kLds + 2 * (2 * BN + BM) * 4;

  const Int8Params& p;
  char* lds;
  int first, last, pitch;
  int64_t m0, n0;
  template <typename Tile>
  FLA_DEVICE void start(Tile& t) const { t.start(pitch, pitch); }
  FLA_DEVICE void at(uint32_t tm, uint32_t n) { m0 = (int64_t)tm * BM, n0 = (int64_t)n * (BN / 2); }
  FLA_DEVICE void source(int s, MatSource* m, MatSource* n) const {
    const int k = s * kSliceBytes;
    m[0] = MatSource{p.x + m0 * pitch + k, p.x + p.M * pitch, pitch - k};
    n[0] = MatSource{p.w + n0 * pitch + k, p.w + p.N * pitch, pitch - k};
  }
  // Biases and scales of the columns, two waves each, as they lie in memory; zeros where there are none.  The third: scales of the rows.
  FLA_DEVICE char* column(int side, int which) const { return lds + Whole::kLds + side * (2 * BN + BM) * 4 + which * BN * 4; }
  FLA_DEVICE void columns(int side) const {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), which = wave >> 1;
    const char* from = (const char*)(which ? (const void*)p.sw : p.bias);
    const int e = which || p.bias_f32 ? 4 : (int)sizeof(O);
    const __amdgpu_buffer_rsrc_t d = MatSource{from + n0 * e, from ? from + (p.N * e + 3) / 4 * 4 : nullptr, 0}.descriptor();   // (whole words)
#pragma unroll
    for (int q = 0; q < BN * 2 / 256; ++q) {
      const int at = ((wave & 1) * (BN * 2 / 256) + q) * 256;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(d, (__attribute__((address_space(3))) void*)(column(side, which) + at), 4, at + lane * 4, 0, 0, 0);
    }
    if (wave * 64 < BM) {
      const __amdgpu_buffer_rsrc_t r = MatSource{(const char*)(p.sx + m0), (const char*)(p.sx + p.M), 0}.descriptor();
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(column(side, 2) + wave * 256), 4, wave * 256 + lane * 4, 0, 0, 0);
    }
  }
  FLA_DEVICE f32x4 bias4(int side, int n) const {
    const char* c = column(side, 0);
    if (p.bias_f32) return *(const f32x4*)(c + n * 4);
    typedef O V4 __attribute__((ext_vector_type(4)));
    const V4 v = *(const V4*)(c + n * sizeof(O));
    return f32x4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
  }
  // 1: every store was made, 16 bytes each, and nothing was loaded
  template <typename Tile>
  FLA_DEVICE int finish(const Tile& t, const typename Tile::acc_t (&acc)[Tile::MT][Tile::NT], int side) const {
    const int lr = t.lane & 31, lh = t.lane >> 5;
    if (p.splits > 1) {   // int8_finish_kernel adds the slices' sums
      int* part = p.part + blockIdx.y * p.M * p.N;
#pragma unroll
      for (int i = 0; i < Tile::MT; ++i)
#pragma unroll
        for (int j = 0; j < Tile::NT; ++j) {
          const i32x16 a = mat_sums<Tile>(acc, i, j);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            typedef int S4 __attribute__((ext_vector_type(4), aligned(4)));
            const int64_t m = m0 + (t.wm * Tile::MT + i) * 32 + lr, n = n0 + (t.wn * Tile::NT + j) * 32 + 8 * q + 4 * lh;
            int* to = part + m * p.N + n;
            if (m < p.M && n + 4 <= p.N) {
              *(S4*)to = S4{a[4 * q], a[4 * q + 1], a[4 * q + 2], a[4 * q + 3]};
            } else if (m < p.M) {
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (n + r < p.N) to[r] = a[4 * q + r];
            }
          }
          mat_piece_end();
        }
      return 0;
    }
    with_this_activation<ACT>(p.act, [&](auto act) {
#pragma unroll
      for (int i = 0; i < Tile::MT; ++i) {
        const int64_t m = m0 + (t.wm * Tile::MT + i) * 32 + lr;
        const float sx = *(const float*)(column(side, 2) + ((t.wm * Tile::MT + i) * 32 + lr) * 4);
#pragma unroll
        for (int j = 0; j < Tile::NT; ++j) {
          // (the residual of 32 columns ahead of their stores: a load waits for every store ahead of it)
          f32x4 res[2][2];
#pragma unroll
          for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int e = 0; e < 2; ++e) res[q][e] = RES ? int8_residual<O>(p, m, n0 + (t.wn * Tile::NT + j) * 32 + 16 * q + 8 * e + 4 * lh) : f32x4{0.f, 0.f, 0.f, 0.f};
          const i32x16 a = mat_sums<Tile>(acc, i, j);
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const int nl = (t.wn * Tile::NT + j) * 32 + 16 * q + 4 * lh;     // of the first run of four; the second is eight further
            float v[2][4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const i32x4 sums = {a[8 * q + 4 * e], a[8 * q + 4 * e + 1], a[8 * q + 4 * e + 2], a[8 * q + 4 * e + 3]};
              int8_values<decltype(act)::value>(sums, sx, *(const f32x4*)(column(side, 1) + (nl + 8 * e) * 4), bias4(side, nl + 8 * e), res[q][e], v[e]);
            }
            if constexpr (sizeof(O) == 2) {
              const i32x4 o = mat_join(pack4<O>(v[0]), pack4<O>(v[1]));
              if (m < p.M) store_piece((O*)p.y + m * p.N, n0 + nl + 4 * lh, p.N, o);
            } else {
              int8_store4<O>(p, m, n0 + nl, v[0]);
              int8_store4<O>(p, m, n0 + nl + 8, v[1]);
            }
            mat_piece_end();
          }
        }
      }
    });
    return sizeof(O) == 2 && !p.res && m0 + BM <= p.M && n0 + Tile::NT * 64 <= p.N;
  }
};

template <typename O, int BM, int BN, int PER_SIMD, bool HALVES, bool RES, int ACT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(PER_SIMD, PER_SIMD))) void int8_tile_kernel(Int8Params p, MatGrid grid) {
  typedef Int8Job<O, BM, BN, HALVES, RES, ACT> Job;
  __shared__ __attribute__((aligned(1024))) char lds[Job::kLds];
  const int pitch = (int)p.K, slices = (pitch + kSliceBytes - 1) / kSliceBytes, per = (slices + p.splits - 1) / p.splits, first = blockIdx.y * per;
  Job job{p, lds, first, first + per < slices ? first + per : slices, pitch, 0, 0};
  mat_run(lds, grid, job);
}

// At most MT x 16 rows of x: sixteen columns of y to a workgroup
template <typename O, int MT, int WAVES, int RING>
__global__ __launch_bounds__(WAVES * 64) void int8_panel_kernel(Int8Params p) {
  typedef MatPanel<int8_t, MT, 1, WAVES, RING> Panel;
  __shared__ __attribute__((aligned(16))) char lds[Panel::kLds];
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int lane = threadIdx.x & 63;
  const char* const w[1] = {p.w + n0 * p.K};
  Panel::run(lds, p.x, p.M, w, p.N - n0, (int)p.K, [&](const typename Panel::acc_t* sums, int j) {
    const int64_t m = j * 16 + (lane & 15), n = n0 + (lane >> 4) * 4;
    f32x4 sw, bias;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      sw[r] = n + r < p.N ? p.sw[n + r] : 0.f;
      bias[r] = int8_bias<O>(p, n + r);
    }
    float v[4];
    const f32x4 res = int8_residual<O>(p, m, n);
    with_activation(p.act, [&](auto act) { int8_values<decltype(act)::value>(sums[0], m < p.M ? p.sx[m] : 0.f, sw, bias, res, v); });
    int8_store4<O>(p, m, n, v);
  });
}

// y from the sums of slices of K: four columns a thread
template <typename O>
__global__ __launch_bounds__(256) void int8_finish_kernel(Int8Params p) {
  const int64_t per = (p.N + 3) / 4, id = (int64_t)blockIdx.x * 256 + threadIdx.x, m = id / per, n = id % per * 4;
  if (m >= p.M) return;
  i32x4 sums = {0, 0, 0, 0};
  f32x4 sw, bias;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    sw[r] = n + r < p.N ? p.sw[n + r] : 0.f;
    bias[r] = int8_bias<O>(p, n + r);
    if (n + r < p.N)
      for (int s = 0; s < p.splits; ++s) sums[r] += p.part[(s * p.M + m) * p.N + n + r];
  }
  float v[4];
  const f32x4 res = int8_residual<O>(p, m, n);
  with_activation(p.act, [&](auto act) { int8_values<decltype(act)::value>(sums, p.sx[m], sw, bias, res, v); });
  int8_store4<O>(p, m, n, v);
}

template <typename O>
int launch_int8(Int8Params& p, hipStream_t st) {
  if (p.M <= kPanelRows) {
    const dim3 grid((unsigned)fla_cdiv(p.N, 16));
    if (p.M <= 16) hipLaunchKernelGGL((int8_panel_kernel<O, 1, 4, 2>), grid, dim3(256), 0, st, p);
    else if (p.M <= 32) hipLaunchKernelGGL((int8_panel_kernel<O, 2, 4, 2>), grid, dim3(256), 0, st, p);
    else if (p.M <= 48) hipLaunchKernelGGL((int8_panel_kernel<O, 3, 4, 2>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((int8_panel_kernel<O, 4, 4, 2>), grid, dim3(256), 0, st, p);
    FLA_CHECK_LAUNCH();
    return FLA_OK;
  }
  const TilePlan plan = plan_int8(p.M, p.N, p.K, sizeof(O) == 2);
  FLA_REQUIRE(plan.splits == 1 || p.part, FLA_E_INVALID);
  p.splits = plan.splits;
  MatGrid g{};
  dim3 grid;
  const int rc = grid_of(plan.kind, fla_cdiv(p.M, kTileM[plan.kind]), fla_cdiv(p.N, kTileN[plan.kind]), p.splits, &g, &grid);
  if (rc != FLA_OK) return rc;
  if (plan.kind == kBig) {
    if constexpr (sizeof(O) == 2)
      for_activation(p.act, [&](auto act) {
        constexpr int A = decltype(act)::value;
        if (p.res) hipLaunchKernelGGL((int8_tile_kernel<O, 256, 256, 1, true, true, A>), grid, dim3(256), 0, st, p, g);
        else hipLaunchKernelGGL((int8_tile_kernel<O, 256, 256, 1, true, false, A>), grid, dim3(256), 0, st, p, g);
        return 0;
      });
  } else if (plan.kind == kMiddle) {
    hipLaunchKernelGGL((int8_tile_kernel<O, 128, 128, 2, false, true, -1>), grid, dim3(256), 0, st, p, g);
  } else {
    hipLaunchKernelGGL((int8_tile_kernel<O, 64, 128, 3, false, true, -1>), grid, dim3(256), 0, st, p, g);
  }
  FLA_CHECK_LAUNCH();
  if (p.splits > 1) {
    hipLaunchKernelGGL((int8_finish_kernel<O>), dim3((unsigned)fla_cdiv(p.M * fla_cdiv(p.N, 4), 256)), dim3(256), 0, st, p);
    FLA_CHECK_LAUNCH();
  }
  return FLA_OK;
}

}  // namespace
