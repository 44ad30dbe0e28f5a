// The gated product of a feed-forward block:   g = x Wg' + bg,   u = x Wu' + bu,   h = act(g) u      x [M,K], Wg, Wu [F,K], act: none, silu, gelu, relu
// One launch on the tiles of matrix_tiles.h.  The rows of the two weights alternate in a tile, 32 of each, so that the lane that holds sums of
// the gate holds those of the same m and n of the other projection, and neither goes through memory.  For the backward g and u are kept in fp32, as they
// are summed: the slope of a gate that fp16 does not hold is right, and dg and du carry their own rounding to 16 bits alone.
// Measured: 8191 x 2048 to 5632 with gelu and biases 356 - 374 us (1.01 - 1.06 PFLOP/s; torch's product alone of that size 395 - 401), with silu and g, u kept 411 - 416 (of which
// the 369 MB of g and u against as much in 16 bits 20 - 30), in integers 202 - 224 (1.7 - 1.87 POP/s).  Its 1408 tiles are five and a half rounds of some 65 us, of which 32 slices at 1.6
// are 51.  What bounds it: matrix instructions are busy in 0.49 of its cycles (0.76 at 8192^3): slices wait for memory, and the ends of tiles
// (activations, stores of 16 bytes a lane that take a row in pieces of 32) have none.
// Of rows in 8-bit integers the sums are exact, and scaled where the biases are added.
#pragma once
#include "linear_epilogue.h"
#include "matrix_panels.h"
#include "matrix_plan.h"
#include "matrix_tiles.h"

namespace {

struct GatedParams {
  const char *x, *wg, *wu;       // 16-bit elements, or 8-bit integers
  const float *sx, *sg, *su;     // scales of rows of 8-bit integers
  const void *bg, *bu;           // [F] or NULL
  void *h;                       // [M,F]
  float *g, *u;                  // [M,ldk], kept for the backward, or NULL
  void* part;                    // sums of slices of K [splits, M, 2, F], fp32 or int32, or NULL
  int64_t M, F, K, ldk;
  int act, bias_f32, splits;
};

template <typename O>
FLA_DEVICE float gated_bias(const void* b, int f32, int64_t n, int64_t F) {
  return !b || n >= F ? 0.f : f32 ? ((const float*)b)[n] : (float)((const O*)b)[n];
}

// T: type of the operands, O: of h; ACT: the activation, or -1 for any (one function that holds all four of a big tile takes the compiler minutes)
template <typename T, typename O, int BM, int BN, bool HALVES, int ACT>
struct GatedJob {
  static constexpr bool INT = sizeof(T) == 1, kHalves = HALVES;
  static constexpr int HN = BN / 2;                     // columns of h
  typedef MatTile<T, BM, BN, 2, false, false, true> Whole;
  typedef MatTile<T, BM, HALVES ? BN / 2 : BN, 2, false, false, true> Half;
  static constexpr int LATER = Whole::MT * Whole::NT;   // stores of h
  static constexpr int kLds = Whole::kLds + 2 * (4 * HN + BM) * 4;

  const GatedParams& p;
  char* lds;
  int first, last, pitch;
  int64_t m0, n0;
  template <typename Tile>
  FLA_DEVICE void start(Tile& t) const { t.start(pitch, pitch); }
  FLA_DEVICE void at(uint32_t tm, uint32_t n) { m0 = (int64_t)tm * BM, n0 = (int64_t)n * (HN / 2); }
  FLA_DEVICE void source(int s, MatSource* m, MatSource* n) const {
    const int k = s * kSliceBytes;
    m[0] = MatSource{p.x + m0 * pitch + k, p.x + p.M * pitch, pitch - k};
    n[0] = MatSource{p.wg + n0 * pitch + k, p.wg + p.F * pitch, pitch - k};
    n[1] = MatSource{p.wu + n0 * pitch + k, p.wu + p.F * pitch, pitch - k};
  }
  // Biases and scales of the columns: a wave each, as they lie in memory; zeros where there are none.  The fifth: scales of the rows.
  FLA_DEVICE char* column(int side, int which) const { return lds + Whole::kLds + side * (4 * HN + BM) * 4 + which * HN * 4; }
  FLA_DEVICE void columns(int side) const {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const char* from = (const char*)(wave == 0 ? p.bg : wave == 1 ? p.bu : wave == 2 ? (const void*)p.sg : (const void*)p.su);
    const int e = wave >= 2 || p.bias_f32 ? 4 : (int)sizeof(O);
    const __amdgpu_buffer_rsrc_t d = MatSource{from + n0 * e, from ? from + (p.F * e + 3) / 4 * 4 : nullptr, 0}.descriptor();   // (whole words)
#pragma unroll
    for (int q = 0; q < HN * 4 / 256; ++q)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(d, (__attribute__((address_space(3))) void*)(column(side, wave) + q * 256), 4, q * 256 + lane * 4, 0, 0, 0);
    if (INT && wave * 64 < BM) {
      const __amdgpu_buffer_rsrc_t r = MatSource{(const char*)(p.sx + m0), (const char*)(p.sx + p.M), 0}.descriptor();
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(column(side, 4) + wave * 256), 4, wave * 256 + lane * 4, 0, 0, 0);
    }
  }
  FLA_DEVICE f32x4 bias4(int side, int which, int n) const {
    const char* c = column(side, which);
    if (p.bias_f32) return *(const f32x4*)(c + n * 4);
    const typename Elem<O>::v4 v = *(const typename Elem<O>::v4*)(c + n * 2);
    return f32x4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
  }
  // 1: every store was made, and only those of h;  2: also those of g and u
  template <typename Tile>
  FLA_DEVICE int finish(const Tile& t, const typename Tile::acc_t (&acc)[Tile::MT][Tile::NT], int side) const {
    constexpr int TN = Tile::NT * 32;      // columns of h of the tile
    const int lr = t.lane & 31, lh = t.lane >> 5;
    const int64_t mw = m0 + t.wm * (BM / 2) + lr;
    if (p.splits > 1) {   // gated_finish_kernel adds the slices' sums
      typedef typename std::conditional<INT, int, float>::type S;
      S* part = (S*)p.part + blockIdx.y * p.M * 2 * p.F;
#pragma unroll
      for (int i = 0; i < Tile::MT; ++i)
#pragma unroll
        for (int j = 0; j < Tile::NT; ++j) {
          const typename Tile::acc_t a = mat_sums<Tile>(acc, i, j);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            typedef S S4 __attribute__((ext_vector_type(4), aligned(4)));
            const int64_t m = mw + i * 32, n = n0 + t.wn * (TN / 2) + j / 2 * 32 + 8 * q + 4 * lh;
            S* to = part + (m * 2 + j % 2) * p.F + n;
            if (m < p.M && n + 4 <= p.F) {
              *(S4*)to = S4{a[4 * q], a[4 * q + 1], a[4 * q + 2], a[4 * q + 3]};
            } else if (m < p.M) {
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (n + r < p.F) to[r] = a[4 * q + r];
            }
          }
          mat_piece_end();
        }
      return 0;
    }
    with_this_activation<ACT>(p.act, [&](auto act) {
#pragma unroll
      for (int i = 0; i < Tile::MT; ++i) {
        const int64_t m = mw + i * 32;
        const float sx = INT ? *(const float*)(column(side, 4) + (t.wm * (BM / 2) + i * 32 + lr) * 4) : 1.f;
#pragma unroll
        for (int h = 0; h < Tile::NT / 2; ++h) {
          const typename Tile::acc_t gs = mat_sums<Tile>(acc, i, 2 * h), us = mat_sums<Tile>(acc, i, 2 * h + 1);
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const int nl = t.wn * (TN / 2) + h * 32 + 16 * q + 4 * lh;     // of the first run of four; the second is eight further
            u32x2 hv[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const f32x4 bg = bias4(side, 0, nl + 8 * e), bu = bias4(side, 1, nl + 8 * e);
              f32x4 sg, su;
              if (INT) sg = *(const f32x4*)(column(side, 2) + (nl + 8 * e) * 4), su = *(const f32x4*)(column(side, 3) + (nl + 8 * e) * 4);
              float g[4], u[4], v[4];
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                g[r] = (float)gs[8 * q + 4 * e + r], u[r] = (float)us[8 * q + 4 * e + r];
                if (INT) g[r] = fmaf(g[r], sx * sg[r], bg[r]), u[r] = fmaf(u[r], sx * su[r], bu[r]);
                else g[r] += bg[r], u[r] += bu[r];
                v[r] = activate_gate<decltype(act)::value>(g[r]) * u[r];
              }
              hv[e] = pack4<O>(v);
              const int64_t n = n0 + nl + 8 * e;
              if (!INT && p.g && m < p.M && n < p.ldk) {     // (ldk is a multiple of 8)
                *(f32x4*)(p.g + m * p.ldk + n) = f32x4{g[0], g[1], g[2], g[3]};
                *(f32x4*)(p.u + m * p.ldk + n) = f32x4{u[0], u[1], u[2], u[3]};
              }
            }
            const i32x4 ho = mat_join(hv[0], hv[1]);
            const int64_t n = n0 + t.wn * (TN / 2) + h * 32 + 16 * q + 8 * lh;
            if (m < p.M) store_piece((O*)p.h + m * p.F, n, p.F, ho);
            mat_piece_end();
          }
        }
      }
    });
    return m0 + BM <= p.M && n0 + TN <= p.F ? (p.g ? 2 : 1) : 0;
  }
};

template <typename T, typename O, int BM, int BN, int PER_SIMD, bool HALVES, int ACT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(PER_SIMD, PER_SIMD))) void gated_tile_kernel(GatedParams p, MatGrid grid) {
  typedef GatedJob<T, O, BM, BN, HALVES, ACT> Job;
  __shared__ __attribute__((aligned(1024))) char lds[Job::kLds];
  const int pitch = (int)(p.K * sizeof(T)), slices = (pitch + kSliceBytes - 1) / kSliceBytes, per = (slices + p.splits - 1) / p.splits;
  const int first = blockIdx.y * per;
  Job job{p, lds, first, first + per < slices ? first + per : slices, pitch, 0, 0};
  mat_run(lds, grid, job);
}

// h (g, u) from the sums of slices of K, added in their order: four columns a thread
template <typename T, typename O>
__global__ __launch_bounds__(256) void gated_finish_kernel(GatedParams p) {
  constexpr bool INT = sizeof(T) == 1;
  typedef typename std::conditional<INT, int, float>::type S;
  typedef S S4 __attribute__((ext_vector_type(4), aligned(4)));
  const int64_t per = (p.ldk + 3) / 4, id = (int64_t)blockIdx.x * 256 + threadIdx.x, m = id / per, n0 = id % per * 4;
  if (m >= p.M) return;
  const bool whole = n0 + 4 <= p.F;
  S4 g = {0, 0, 0, 0}, u = {0, 0, 0, 0};
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    const S* from = (const S*)p.part + (s * p.M + m) * 2 * p.F + n0;
    if (whole) {
      g += *(const S4*)from, u += *(const S4*)(from + p.F);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n0 + i < p.F) g[i] += from[i], u[i] += from[p.F + i];
    }
  }
  const float sx = INT ? p.sx[m] : 1.f;
  float gf[4], uf[4], v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t n = n0 + i;
    const float bg = gated_bias<O>(p.bg, p.bias_f32, n, p.F), bu = gated_bias<O>(p.bu, p.bias_f32, n, p.F);
    gf[i] = INT ? fmaf((float)g[i], n < p.F ? sx * p.sg[n] : 0.f, bg) : (float)g[i] + bg;
    uf[i] = INT ? fmaf((float)u[i], n < p.F ? sx * p.su[n] : 0.f, bu) : (float)u[i] + bu;
  }
  with_activation(p.act, [&](auto act) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = activate_gate<decltype(act)::value>(gf[i]) * uf[i];
  });
  O* h = (O*)p.h + m * p.F + n0;
  if (whole) {
    typedef u32x2 any __attribute__((aligned(2)));
    *(any*)h = pack4<O>(v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n0 + i < p.F) h[i] = (O)v[i];
  }
  if (!INT && p.g && n0 < p.ldk) {     // (ldk is a multiple of 8)
    *(f32x4*)(p.g + m * p.ldk + n0) = f32x4{gf[0], gf[1], gf[2], gf[3]};
    *(f32x4*)(p.u + m * p.ldk + n0) = f32x4{uf[0], uf[1], uf[2], uf[3]};
  }
}

// At most MT x 16 rows of x: sixteen columns of h to a workgroup
template <typename T, typename O, int MT, int WAVES, int RING>
__global__ __launch_bounds__(WAVES * 64) void gated_panel_kernel(GatedParams p) {
  typedef MatPanel<T, MT, 2, WAVES, RING> Panel;
  constexpr bool INT = sizeof(T) == 1;
  __shared__ __attribute__((aligned(16))) char lds[Panel::kLds];
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int pitch = (int)(p.K * sizeof(T)), lane = threadIdx.x & 63;
  const char* const w[2] = {p.wg + n0 * pitch, p.wu + n0 * pitch};
  Panel::run(lds, p.x, p.M, w, p.F - n0, pitch, [&](const typename Panel::acc_t* sums, int j) {
    const int64_t m = j * 16 + (lane & 15), n = n0 + (lane >> 4) * 4;
    if (m >= p.M) return;
    const float sx = INT ? p.sx[m] : 1.f;
    float g[4], u[4], v[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float bg = gated_bias<O>(p.bg, p.bias_f32, n + r, p.F), bu = gated_bias<O>(p.bu, p.bias_f32, n + r, p.F);
      g[r] = INT ? fmaf((float)sums[0][r], n + r < p.F ? sx * p.sg[n + r] : 0.f, bg) : (float)sums[0][r] + bg;
      u[r] = INT ? fmaf((float)sums[1][r], n + r < p.F ? sx * p.su[n + r] : 0.f, bu) : (float)sums[1][r] + bu;
    }
    with_activation(p.act, [&](auto act) {
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = activate_gate<decltype(act)::value>(g[r]) * u[r];
    });
    O* h = (O*)p.h + m * p.F + n;
    if (n + 4 <= p.F) {
      typedef u32x2 any __attribute__((aligned(2)));
      *(any*)h = pack4<O>(v);
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (n + r < p.F) h[r] = (O)v[r];
    }
    if (!INT && p.g && n < p.ldk) {     // (ldk is a multiple of 8)
      *(f32x4*)(p.g + m * p.ldk + n) = f32x4{g[0], g[1], g[2], g[3]};
      *(f32x4*)(p.u + m * p.ldk + n) = f32x4{u[0], u[1], u[2], u[3]};
    }
  });
}

template <typename T, typename O>
int launch_forward(const GatedParams& p, TileKind kind, hipStream_t st) {
  MatGrid g{};
  dim3 grid;
  const int rc = grid_of(kind, fla_cdiv(p.M, kTileM[kind]), fla_cdiv(p.F, kTileN[kind] / 2), p.splits, &g, &grid);
  if (rc != FLA_OK) return rc;
  if (kind == kBig)
    for_activation(p.act, [&](auto act) {
      hipLaunchKernelGGL((gated_tile_kernel<T, O, 256, 256, 1, true, decltype(act)::value>), grid, dim3(256), 0, st, p, g);
      return 0;
    });
  else if (kind == kMiddle) hipLaunchKernelGGL((gated_tile_kernel<T, O, 128, 128, 2, false, -1>), grid, dim3(256), 0, st, p, g);
  else hipLaunchKernelGGL((gated_tile_kernel<T, O, 64, 128, 3, false, -1>), grid, dim3(256), 0, st, p, g);
  FLA_CHECK_LAUNCH();
  if (p.splits > 1) {
    hipLaunchKernelGGL((gated_finish_kernel<T, O>), dim3((unsigned)fla_cdiv(p.M * fla_cdiv(p.ldk, 4), 256)), dim3(256), 0, st, p);
    FLA_CHECK_LAUNCH();
  }
  return FLA_OK;
}
template <typename T, typename O>
int launch_panel(const GatedParams& p, hipStream_t st) {
  const int64_t grid = fla_cdiv(p.F, 16);
  if (p.M <= 16) hipLaunchKernelGGL((gated_panel_kernel<T, O, 1, 4, 2>), dim3((unsigned)grid), dim3(256), 0, st, p);
  else if (p.M <= 32) hipLaunchKernelGGL((gated_panel_kernel<T, O, 2, 4, 2>), dim3((unsigned)grid), dim3(256), 0, st, p);
  else if (p.M <= 48) hipLaunchKernelGGL((gated_panel_kernel<T, O, 3, 4, 2>), dim3((unsigned)grid), dim3(256), 0, st, p);
  else hipLaunchKernelGGL((gated_panel_kernel<T, O, 4, 4, 2>), dim3((unsigned)grid), dim3(256), 0, st, p);
  FLA_CHECK_LAUNCH();
  return FLA_OK;
}
template <typename T, typename O>
int gated_forward(GatedParams& p, hipStream_t st) {
  if (p.M <= kPanelRows) return launch_panel<T, O>(p, st);
  const TilePlan plan = plan_gated(p.M, p.F, p.K * sizeof(T));
  FLA_REQUIRE(plan.splits == 1 || p.part, FLA_E_INVALID);
  p.splits = plan.splits;
  return launch_forward<T, O>(p, plan.kind, st);
}

}  // namespace
