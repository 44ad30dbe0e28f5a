// The gated product of a feed-forward block, and its gradients:
//   g = x Wg' + bg,   u = x Wu' + bu,   h = act(g) u            x [M,K], Wg, Wu [F,K], act: none, silu, gelu, relu
//   dg = dh u act'(g),   du = dh act(g),   dx = dg Wg + du Wu,   dWg = dg' x,   dWu = du' x,   dbg, dbu: column sums of dg and du
// Forward: one launch on the tiles of matrix_tiles.h.  The rows of the two weights alternate in a tile, 32 of each, so that the lane that holds sums of
// the gate holds those of the same m and n of the other projection, and neither goes through memory.  For the backward g and u are kept in the
// operands' type: dg and du then carry that rounding beside their own, each half a step.  h itself comes from the fp32 sums.
// Backward: dg and du in one pass over dh, g and u (HBM-bound), with the column sums of the biases' gradients; dx as one product over both halves of the
// contraction, its second operand strided in memory; the weights' gradients as one launch of products with both operands strided.
#include "linear_epilogue.h"
#include "matrix_panels.h"
#include "matrix_plan.h"
#include "matrix_tiles.h"
#include "row_vec.h"

namespace {

struct GatedParams {
  const char *x, *wg, *wu;       // 16-bit elements, or 8-bit integers
  const float *sx, *sg, *su;     // scales of rows of 8-bit integers
  const void *bg, *bu;           // [F] or NULL
  void *h;                       // [M,F]
  void *g, *u;                   // [M,ldk], kept for the backward, or NULL
  void* part;                    // sums of slices of K [splits, M, 2, F], fp32 or int32, or NULL
  int64_t M, F, K, ldk;
  int act, bias_f32, splits;
  bool wide;                     // rows of h can be written 16 bytes at a time
};

template <typename O>
FLA_DEVICE float gated_bias(const void* b, int f32, int64_t n, int64_t F) {
  return !b || n >= F ? 0.f : f32 ? ((const float*)b)[n] : (float)((const O*)b)[n];
}

// T: type of the operands, O: of h
template <typename T, typename O, int BM, int BN, bool HALVES>
struct GatedJob {
  static constexpr bool INT = sizeof(T) == 1, kHalves = HALVES;
  static constexpr int HN = BN / 2;                     // columns of h
  typedef MatTile<T, BM, BN, 2, false, false, true> Whole;
  typedef MatTile<T, BM, HALVES ? BN / 2 : BN, 2, false, false, true> Half;
  static constexpr int LATER = Whole::MT * Whole::NT;   // stores of h
  static constexpr int kLds = Whole::kLds + 2 * 4 * HN * 4;

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
  // Biases and scales of the columns: a wave each, as they lie in memory; zeros where there are none
  FLA_DEVICE char* column(int side, int which) const { return lds + Whole::kLds + (side * 4 + which) * HN * 4; }
  FLA_DEVICE void columns(int side) const {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const char* from = (const char*)(wave == 0 ? p.bg : wave == 1 ? p.bu : wave == 2 ? (const void*)p.sg : (const void*)p.su);
    const int e = wave >= 2 || p.bias_f32 ? 4 : (int)sizeof(O);
    const __amdgpu_buffer_rsrc_t d = MatSource{from + n0 * e, from ? from + (p.F * e + 3) / 4 * 4 : nullptr, 0}.descriptor();   // (whole words)
#pragma unroll
    for (int q = 0; q < HN * 4 / 256; ++q)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(d, (__attribute__((address_space(3))) void*)(column(side, wave) + q * 256), 4, q * 256 + lane * 4, 0, 0, 0);
  }
  FLA_DEVICE f32x4 bias4(int side, int which, int n) const {
    const char* c = column(side, which);
    if (p.bias_f32) return *(const f32x4*)(c + n * 4);
    const typename Elem<O>::v4 v = *(const typename Elem<O>::v4*)(c + n * 2);
    return f32x4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
  }
  // true: every store was made, and only those of h
  template <typename Tile>
  FLA_DEVICE bool finish(const Tile& t, const typename Tile::acc_t (&acc)[Tile::MT][Tile::NT], int side) const {
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
      return false;
    }
    with_activation(p.act, [&](auto act) {
#pragma unroll
      for (int i = 0; i < Tile::MT; ++i) {
        const int64_t m = mw + i * 32;
        const float sx = INT && m < p.M ? p.sx[m] : 1.f;
#pragma unroll
        for (int h = 0; h < Tile::NT / 2; ++h) {
          const typename Tile::acc_t gs = mat_sums<Tile>(acc, i, 2 * h), us = mat_sums<Tile>(acc, i, 2 * h + 1);
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const int nl = t.wn * (TN / 2) + h * 32 + 16 * q + 4 * lh;     // of the first run of four; the second is eight further
            u32x2 hv[2], gv[2], uv[2];
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
              hv[e] = pack4<O>(v), gv[e] = pack4<O>(g), uv[e] = pack4<O>(u);
            }
            const i32x4 ho = mat_join(hv[0], hv[1]);
            const int64_t n = n0 + t.wn * (TN / 2) + h * 32 + 16 * q + 8 * lh;
            if (m < p.M) store_piece((O*)p.h + m * p.F, n, p.F, p.wide, ho);
            if (!INT && p.g) {
              const i32x4 go = mat_join(gv[0], gv[1]), uo = mat_join(uv[0], uv[1]);
              if (m < p.M) {
                store_piece((O*)p.g + m * p.ldk, n, p.ldk, true, go);
                store_piece((O*)p.u + m * p.ldk, n, p.ldk, true, uo);
              }
            }
            mat_piece_end();
          }
        }
      }
    });
    return !INT && !p.g && p.wide && m0 + BM <= p.M && n0 + TN <= p.F;
  }
};

template <typename T, typename O, int BM, int BN, int PER_SIMD, bool HALVES>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(PER_SIMD, PER_SIMD))) void gated_tile_kernel(GatedParams p, MatGrid grid) {
  typedef GatedJob<T, O, BM, BN, HALVES> Job;
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
  const int64_t per = (p.ldk + 3) / 4, id = (int64_t)blockIdx.x * 256 + threadIdx.x, m = id / per, n0 = id % per * 4;
  if (m >= p.M) return;
  const float sx = INT ? p.sx[m] : 1.f;
  with_activation(p.act, [&](auto act) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t n = n0 + i;
      S g = 0, u = 0;
      if (n < p.F)
        for (int s = 0; s < p.splits; ++s) {
          const S* from = (const S*)p.part + (s * p.M + m) * 2 * p.F + n;
          g += from[0], u += from[p.F];
        }
      const float bg = gated_bias<O>(p.bg, p.bias_f32, n, p.F), bu = gated_bias<O>(p.bu, p.bias_f32, n, p.F);
      const float gf = INT ? fmaf((float)g, n < p.F ? sx * p.sg[n] : 0.f, bg) : (float)g + bg;
      const float uf = INT ? fmaf((float)u, n < p.F ? sx * p.su[n] : 0.f, bu) : (float)u + bu;
      if (n < p.F) ((O*)p.h)[m * p.F + n] = (O)(activate_gate<decltype(act)::value>(gf) * uf);
      if (!INT && p.g && n < p.ldk) ((O*)p.g)[m * p.ldk + n] = (O)gf, ((O*)p.u)[m * p.ldk + n] = (O)uf;
    }
  });
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
    if (p.wide && n + 4 <= p.F) {
      *(u32x2*)h = pack4<O>(v);
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (n + r < p.F) h[r] = (O)v[r];
    }
    if (!INT && p.g && n < p.ldk) {     // (ldk is a multiple of 8)
      *(u32x2*)((O*)p.g + m * p.ldk + n) = pack4<O>(g);
      *(u32x2*)((O*)p.u + m * p.ldk + n) = pack4<O>(u);
    }
  });
}

// ------------------------------------------------------------------------------------------------ backward
struct GatedBwdParams {
  const void *dh, *g, *u;     // [M,F], [M,ld], [M,ld]
  void *dg, *du;              // [M,ld]: columns behind F are zeros
  float *pg, *pu;             // partial sums [gridDim.y, F] or NULL
  int64_t M, F, ld, rows;     // rows: of a workgroup
  int act;
};

// 512 columns, eight a thread, of `rows` rows, four at a time
template <typename T>
__global__ __launch_bounds__(256) void gated_bwd_kernel(GatedBwdParams p) {
  __shared__ float sum[2][4][512];
  const int cl = threadIdx.x & 63, rl = threadIdx.x >> 6;
  const int64_t col = (int64_t)blockIdx.x * 512 + cl * 8, first = (int64_t)blockIdx.y * p.rows;
  const int64_t end = first + p.rows < p.M ? first + p.rows : p.M;
  const int valid = col >= p.ld ? 0 : p.F - col < 8 ? (int)(p.F - col) : 8;    // (col < ld: F - col > 0, ld being F rounded up to 8)
  float sg[8], su[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) sg[i] = su[i] = 0.f;
  with_activation(p.act, [&](auto act) {
    if (valid > 0)
#pragma unroll 2
      for (int64_t m = first + rl; m < end; m += 4) {
        float d[8], g[8], u[8];
        Row8<T>::unpack(load_raw8<T, false>((const T*)p.dh + m * p.F + col, valid), d);
        Row8<T>::load((const T*)p.g + m * p.ld + col, g);
        Row8<T>::load((const T*)p.u + m * p.ld + col, u);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float slope;
          const float a = activate_gate<decltype(act)::value>(g[i], &slope);
          g[i] = i < valid ? d[i] * u[i] * slope : 0.f;
          u[i] = i < valid ? d[i] * a : 0.f;
          sg[i] += g[i], su[i] += u[i];
        }
        Row8<T>::store((T*)p.dg + m * p.ld + col, g);
        Row8<T>::store((T*)p.du + m * p.ld + col, u);
      }
  });
  if (!p.pg && !p.pu) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) sum[0][rl][cl * 8 + i] = sg[i], sum[1][rl][cl * 8 + i] = su[i];
  __syncthreads();
  for (int k = threadIdx.x; k < 1024; k += 256) {
    const int c = k & 511, which = k >> 9;
    const int64_t n = (int64_t)blockIdx.x * 512 + c;
    float* part = which ? p.pu : p.pg;
    if (part && n < p.F) part[blockIdx.y * p.F + n] = ((sum[which][0][c] + sum[which][1][c]) + sum[which][2][c]) + sum[which][3][c];
  }
}

struct GradParams {
  const char *dg, *du;       // [M,ld]
  const char *a, *b;         // dx: Wg, Wu [F,K];  weights' gradients: x [M,K], -
  void *y, *y2;              // dx [M,K];  dWg, dWu [F,K], either may be NULL
  float* part;               // sums of slices [splits, (2,) rows, K], or NULL
  int64_t M, F, K, ld;
  int splits;
};

// A tile of a gradient of `rows` rows of K elements; true: every store was made, 16 bytes each
template <typename T, typename Tile>
FLA_DEVICE bool grad_store(const Tile& t, const typename Tile::acc_t (&acc)[Tile::MT][Tile::NT], T* y, float* part, int64_t m0, int64_t n0, int64_t rows, int64_t K) {
  const int lr = t.lane & 31, lh = t.lane >> 5;
#pragma unroll
  for (int i = 0; i < Tile::MT; ++i) {
    const int64_t m = m0 + (t.wm * Tile::MT + i) * 32 + lr;
#pragma unroll
    for (int j = 0; j < Tile::NT; ++j) {
      const int64_t n = n0 + (t.wn * Tile::NT + j) * 32;
      const typename Tile::acc_t v = mat_sums<Tile>(acc, i, j);
      if (part) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (m < rows && n + 8 * q + 4 * lh < K)
            *(f32x4*)(part + m * K + n + 8 * q + 4 * lh) = f32x4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
      } else {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          float a[4], b[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) a[r] = v[8 * q + r], b[r] = v[8 * q + 4 + r];
          const i32x4 o = mat_join(pack4<T>(a), pack4<T>(b));
          if (m < rows && n + 16 * q + 8 * lh < K) *(i32x4*)(y + m * K + n + 16 * q + 8 * lh) = o;      // (K is a multiple of 8)
        }
      }
      mat_piece_end();
    }
  }
  return !part && m0 + Tile::MT * 64 <= rows && n0 + Tile::NT * 64 <= K;
}

// dx = dg Wg + du Wu: the slices of the first product, then those of the second
template <typename T, int BM, int BN, bool HALVES>
struct DxJob {
  static constexpr bool kHalves = HALVES;
  typedef MatTile<T, BM, BN, 2, false, true> Whole;
  typedef MatTile<T, BM, HALVES ? BN / 2 : BN, 2, false, true> Half;
  static constexpr int LATER = Whole::MT * Whole::NT * 2, kLds = Whole::kLds;
  const GradParams& p;
  int first, last, each;     // each: slices of one of the products
  int64_t m0, n0;
  template <typename Tile>
  FLA_DEVICE void start(Tile& t) const { t.start((uint32_t)(p.ld * 2), (uint32_t)(p.K * 2)); }
  FLA_DEVICE void at(uint32_t tm, uint32_t n) { m0 = (int64_t)tm * BM, n0 = (int64_t)n * (BN / 2); }
  FLA_DEVICE void columns(int) const {}
  FLA_DEVICE void source(int s, MatSource* m, MatSource* n) const {
    const bool second = s >= each;
    const int k = (second ? s - each : s) * kSliceBytes, pitch = (int)(p.ld * 2);
    const char *d = second ? p.du : p.dg, *w = second ? p.b : p.a;
    m[0] = MatSource{d + m0 * pitch + k, d + p.M * pitch, pitch - k};
    n[0] = MatSource{w + n0 * 2 + (int64_t)(k / 2) * (p.K * 2), w + p.F * p.K * 2, 0};
  }
  template <typename Tile>
  FLA_DEVICE bool finish(const Tile& t, const typename Tile::acc_t (&acc)[Tile::MT][Tile::NT], int) const {
    return grad_store(t, acc, (T*)p.y, p.splits > 1 ? p.part + blockIdx.y * p.M * p.K : nullptr, m0, n0, p.M, p.K);
  }
};
template <typename T, int BM, int BN, int PER_SIMD, bool HALVES>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(PER_SIMD, PER_SIMD))) void gated_dx_kernel(GradParams p, MatGrid grid) {
  typedef DxJob<T, BM, BN, HALVES> Job;
  __shared__ __attribute__((aligned(1024))) char lds[Job::kLds];
  const int each = (int)((p.ld * 2 + kSliceBytes - 1) / kSliceBytes), per = (2 * each + p.splits - 1) / p.splits, first = blockIdx.y * per;
  Job job{p, first, first + per < 2 * each ? first + per : 2 * each, each, 0, 0};
  mat_run(lds, grid, job);
}

// dWg = dg' x and dWu = du' x, the rows of tiles of the one and then those of the other (or one of them alone)
template <typename T, int BM, int BN, bool HALVES>
struct DwJob {
  static constexpr bool kHalves = HALVES;
  typedef MatTile<T, BM, BN, 2, true, true> Whole;
  typedef MatTile<T, BM, HALVES ? BN / 2 : BN, 2, true, true> Half;
  static constexpr int LATER = Whole::MT * Whole::NT * 2, kLds = Whole::kLds;
  const GradParams& p;
  int first, last;
  uint32_t rows;      // of tiles of one weight
  bool up;
  int64_t m0, n0;
  template <typename Tile>
  FLA_DEVICE void start(Tile& t) const { t.start((uint32_t)(p.ld * 2), (uint32_t)(p.K * 2)); }
  FLA_DEVICE void at(uint32_t tm, uint32_t n) {
    up = !p.y || tm >= rows;
    m0 = (int64_t)(tm >= rows ? tm - rows : tm) * BM, n0 = (int64_t)n * (BN / 2);
  }
  FLA_DEVICE void columns(int) const {}
  FLA_DEVICE void source(int s, MatSource* m, MatSource* n) const {
    const int64_t dp = p.ld * 2, xp = p.K * 2;
    const char* d = up ? p.du : p.dg;
    m[0] = MatSource{d + m0 * 2 + (int64_t)s * 64 * dp, d + p.M * dp, 0};
    n[0] = MatSource{p.a + n0 * 2 + (int64_t)s * 64 * xp, p.a + p.M * xp, 0};
  }
  template <typename Tile>
  FLA_DEVICE bool finish(const Tile& t, const typename Tile::acc_t (&acc)[Tile::MT][Tile::NT], int) const {
    const bool second = up && p.y;
    return grad_store(t, acc, (T*)(up ? p.y2 : p.y), p.splits > 1 ? p.part + ((second ? p.splits : 0) + (int64_t)blockIdx.y) * p.F * p.K : nullptr, m0, n0, p.F, p.K);
  }
};
template <typename T, int BM, int BN, int PER_SIMD, bool HALVES>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(PER_SIMD, PER_SIMD))) void gated_dw_kernel(GradParams p, MatGrid grid) {
  typedef DwJob<T, BM, BN, HALVES> Job;
  __shared__ __attribute__((aligned(1024))) char lds[Job::kLds];
  const int slices = (int)((p.M + 63) / 64), per = (slices + p.splits - 1) / p.splits, first = blockIdx.y * per;
  Job job{p, first, first + per < slices ? first + per : slices, (uint32_t)((p.F + BM - 1) / BM), false, 0, 0};
  mat_run(lds, grid, job);
}

// the sums of slices, added in their order: four elements a thread
template <typename T>
__global__ __launch_bounds__(256) void grad_finish_kernel(const float* part, T* y, T* y2, int64_t n, int splits) {
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= n) return;
  const float* from = part + (int64_t)blockIdx.y * splits * n + at;
  f32x4 v = *(const f32x4*)from;
  for (int s = 1; s < splits; ++s) v += *(const f32x4*)(from + s * n);
  typename Elem<T>::v4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = (T)v[i];
  *(typename Elem<T>::v4*)((blockIdx.y || !y ? y2 : y) + at) = o;
}

// ------------------------------------------------------------------------------------------------ host
TilePlan plan_dx(int64_t M, int64_t F, int64_t K) { return plan_tiles(M, K, 2 * fla_cdiv(F * 2, kSliceBytes), 1); }
TilePlan plan_dw(int64_t M, int64_t F, int64_t K, int batch) { return plan_tiles(F, K, fla_cdiv(M, 64), batch); }

template <typename T, typename O>
int launch_forward(const GatedParams& p, TileKind kind, hipStream_t st) {
  MatGrid g{};
  dim3 grid;
  const int rc = grid_of(kind, fla_cdiv(p.M, kTileM[kind]), fla_cdiv(p.F, kTileN[kind] / 2), p.splits, &g, &grid);
  if (rc != FLA_OK) return rc;
  if (kind == kBig) hipLaunchKernelGGL((gated_tile_kernel<T, O, 256, 256, 1, true>), grid, dim3(256), 0, st, p, g);
  else if (kind == kMiddle) hipLaunchKernelGGL((gated_tile_kernel<T, O, 128, 128, 2, false>), grid, dim3(256), 0, st, p, g);
  else hipLaunchKernelGGL((gated_tile_kernel<T, O, 64, 128, 3, false>), grid, dim3(256), 0, st, p, g);
  FLA_CHECK_LAUNCH();
  if (p.splits > 1) {
    hipLaunchKernelGGL((gated_finish_kernel<T, O>), dim3((unsigned)fla_cdiv(p.M * fla_cdiv(p.ldk, 4), 256)), dim3(256), 0, st, p);
    FLA_CHECK_LAUNCH();
  }
  return FLA_OK;
}
template <typename T>
int launch_dx(const GradParams& p, TileKind kind, hipStream_t st) {
  MatGrid g{};
  dim3 grid;
  const int rc = grid_of(kind, fla_cdiv(p.M, kTileM[kind]), fla_cdiv(p.K, kTileN[kind]), p.splits, &g, &grid);
  if (rc != FLA_OK) return rc;
  if (kind == kBig) hipLaunchKernelGGL((gated_dx_kernel<T, 256, 256, 1, true>), grid, dim3(256), 0, st, p, g);
  else if (kind == kMiddle) hipLaunchKernelGGL((gated_dx_kernel<T, 128, 128, 2, false>), grid, dim3(256), 0, st, p, g);
  else hipLaunchKernelGGL((gated_dx_kernel<T, 64, 128, 3, false>), grid, dim3(256), 0, st, p, g);
  FLA_CHECK_LAUNCH();
  if (p.splits > 1) {
    const int64_t n = p.M * p.K;
    hipLaunchKernelGGL((grad_finish_kernel<T>), dim3((unsigned)fla_cdiv(n, 1024)), dim3(256), 0, st, p.part, (T*)p.y, (T*)p.y, n, p.splits);
    FLA_CHECK_LAUNCH();
  }
  return FLA_OK;
}
template <typename T>
int launch_dw(const GradParams& p, TileKind kind, hipStream_t st) {
  const unsigned batch = p.y && p.y2 ? 2 : 1;
  MatGrid g{};
  dim3 grid;
  const int rc = grid_of(kind, batch * fla_cdiv(p.F, kTileM[kind]), fla_cdiv(p.K, kTileN[kind]), p.splits, &g, &grid);
  if (rc != FLA_OK) return rc;
  if (kind == kBig) hipLaunchKernelGGL((gated_dw_kernel<T, 256, 256, 1, true>), grid, dim3(256), 0, st, p, g);
  else if (kind == kMiddle) hipLaunchKernelGGL((gated_dw_kernel<T, 128, 128, 2, false>), grid, dim3(256), 0, st, p, g);
  else hipLaunchKernelGGL((gated_dw_kernel<T, 64, 128, 3, false>), grid, dim3(256), 0, st, p, g);
  FLA_CHECK_LAUNCH();
  if (p.splits > 1) {
    const int64_t n = p.F * p.K;
    hipLaunchKernelGGL((grad_finish_kernel<T>), dim3((unsigned)fla_cdiv(n, 1024), batch), dim3(256), 0, st, p.part, (T*)p.y, (T*)p.y2, n, p.splits);
    FLA_CHECK_LAUNCH();
  }
  return FLA_OK;
}

// Up to this many rows of x go to the panels
constexpr int64_t kPanelRows = 64;
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
TilePlan plan_gated(int64_t M, int64_t F, int64_t row_bytes) { return plan_tiles(M, 2 * F, fla_cdiv(row_bytes, kSliceBytes), 1); }
template <typename T, typename O>
int gated_forward(GatedParams& p, hipStream_t st) {
  if (p.M <= kPanelRows) return launch_panel<T, O>(p, st);
  const TilePlan plan = plan_gated(p.M, p.F, p.K * sizeof(T));
  FLA_REQUIRE(plan.splits == 1 || p.part, FLA_E_INVALID);
  p.splits = plan.splits;
  return launch_forward<T, O>(p, plan.kind, st);
}

}  // namespace

extern "C" int fla_gated_linear_splits(int64_t M, int64_t F, int64_t K, int element_bytes) {
  return M <= kPanelRows || F <= 0 || K <= 0 ? 1 : plan_gated(M, F, K * element_bytes).splits;
}

extern "C" int fla_gated_linear_fwd(const void* x, const void* gate_weight, const void* up_weight, const void* gate_bias, const void* up_bias,
                                    int bias_dtype, void* h, void* gate_out, void* up_out, int64_t ld, int64_t M, int64_t F, int64_t K,
                                    int activation, int dtype, void* workspace, fla_stream_t stream) {
  FLA_REQUIRE(x && gate_weight && up_weight && h && (!gate_out == !up_out) && M >= 0 && F > 0 && K > 0, FLA_E_INVALID);
  FLA_REQUIRE(activation >= FLA_ACT_NONE && activation <= FLA_ACT_RELU, FLA_E_INVALID);
  FLA_REQUIRE(dtype == FLA_BF16 || dtype == FLA_F16, FLA_E_UNSUPPORTED);
  FLA_REQUIRE((!gate_bias && !up_bias) || bias_dtype == dtype || bias_dtype == FLA_F32, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(sizes_ok(M, F, K) && K % 8 == 0, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(!gate_out || (ld >= F && ld % 8 == 0 && ld < F + 8), FLA_E_UNSUPPORTED);
  FLA_REQUIRE(aligned16({x, gate_weight, up_weight, gate_out, up_out, workspace}) && aligned4({gate_bias, up_bias}), FLA_E_ALIGNMENT);
  if (M == 0) return FLA_OK;
  GatedParams p{};
  p.x = (const char*)x, p.wg = (const char*)gate_weight, p.wu = (const char*)up_weight, p.bg = gate_bias, p.bu = up_bias, p.h = h;
  p.g = gate_out, p.u = up_out, p.part = workspace, p.M = M, p.F = F, p.K = K, p.ldk = gate_out ? ld : (F + 7) / 8 * 8;
  p.act = activation, p.bias_f32 = bias_dtype == FLA_F32, p.wide = F % 8 == 0 && aligned16({h});
  hipStream_t st = (hipStream_t)stream;
  return dtype == FLA_BF16 ? gated_forward<bf16, bf16>(p, st) : gated_forward<f16, f16>(p, st);
}

extern "C" int fla_int8_gated_linear_fwd(const void* x, const float* x_scale, const void* gate_weight, const float* gate_scale, const void* up_weight,
                                         const float* up_scale, const void* gate_bias, const void* up_bias, int bias_dtype, void* h, int64_t M,
                                         int64_t F, int64_t K, int activation, int dtype, void* workspace, fla_stream_t stream) {
  FLA_REQUIRE(x && x_scale && gate_weight && gate_scale && up_weight && up_scale && h && M >= 0 && F > 0 && K > 0, FLA_E_INVALID);
  FLA_REQUIRE(activation >= FLA_ACT_NONE && activation <= FLA_ACT_RELU, FLA_E_INVALID);
  FLA_REQUIRE(dtype == FLA_BF16 || dtype == FLA_F16, FLA_E_UNSUPPORTED);
  FLA_REQUIRE((!gate_bias && !up_bias) || bias_dtype == dtype || bias_dtype == FLA_F32, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(sizes_ok(M, F, K) && K % 16 == 0 && K <= FLA_INT8_MAX_K, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(aligned16({x, gate_weight, up_weight, workspace}) && aligned4({gate_bias, up_bias}), FLA_E_ALIGNMENT);
  if (M == 0) return FLA_OK;
  GatedParams p{};
  p.x = (const char*)x, p.wg = (const char*)gate_weight, p.wu = (const char*)up_weight, p.sx = x_scale, p.sg = gate_scale, p.su = up_scale;
  p.bg = gate_bias, p.bu = up_bias, p.h = h, p.part = workspace, p.M = M, p.F = F, p.K = K, p.ldk = (F + 7) / 8 * 8;
  p.act = activation, p.bias_f32 = bias_dtype == FLA_F32, p.wide = F % 8 == 0 && aligned16({h});
  hipStream_t st = (hipStream_t)stream;
  return dtype == FLA_BF16 ? gated_forward<int8_t, bf16>(p, st) : gated_forward<int8_t, f16>(p, st);
}

extern "C" int fla_gated_linear_bwd_rows(int64_t M) { return M <= 0 ? 1 : (int)(fla_cdiv(M, 256) < 32 ? 32 : fla_cdiv(M, 256)); }

extern "C" int fla_gated_linear_bwd_gate(const void* dh, const void* gate, const void* up, void* dgate, void* dup, float* dgate_bias_partial,
                                         float* dup_bias_partial, int64_t ld, int64_t M, int64_t F, int activation, int dtype,
                                         fla_stream_t stream) {
  FLA_REQUIRE(dh && gate && up && dgate && dup && M >= 0 && F > 0, FLA_E_INVALID);
  FLA_REQUIRE(activation >= FLA_ACT_NONE && activation <= FLA_ACT_RELU, FLA_E_INVALID);
  FLA_REQUIRE(dtype == FLA_BF16 || dtype == FLA_F16, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(sizes_ok(M, F, 1) && ld >= F && ld % 8 == 0 && ld < F + 8, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(aligned16({gate, up, dgate, dup}), FLA_E_ALIGNMENT);
  if (M == 0) return FLA_OK;
  GatedBwdParams p{};
  p.dh = dh, p.g = gate, p.u = up, p.dg = dgate, p.du = dup, p.pg = dgate_bias_partial, p.pu = dup_bias_partial, p.M = M, p.F = F, p.ld = ld;
  p.act = activation, p.rows = fla_gated_linear_bwd_rows(M);
  const dim3 grid((unsigned)fla_cdiv(ld, 512), (unsigned)fla_cdiv(M, p.rows));
  hipStream_t st = (hipStream_t)stream;
  if (dtype == FLA_BF16) hipLaunchKernelGGL((gated_bwd_kernel<bf16>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((gated_bwd_kernel<f16>), grid, dim3(256), 0, st, p);
  FLA_CHECK_LAUNCH();
  return FLA_OK;
}

extern "C" int fla_gated_linear_bwd_dx_splits(int64_t M, int64_t F, int64_t K) { return M <= 0 || F <= 0 || K <= 0 ? 1 : plan_dx(M, F, K).splits; }

extern "C" int fla_gated_linear_bwd_dx(const void* dgate, const void* dup, const void* gate_weight, const void* up_weight, void* dx, int64_t ld,
                                       int64_t M, int64_t F, int64_t K, int dtype, float* workspace, fla_stream_t stream) {
  FLA_REQUIRE(dgate && dup && gate_weight && up_weight && dx && M >= 0 && F > 0 && K > 0, FLA_E_INVALID);
  FLA_REQUIRE(dtype == FLA_BF16 || dtype == FLA_F16, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(sizes_ok(M, F, K) && K % 8 == 0 && ld >= F && ld % 8 == 0 && ld < F + 8, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(aligned16({dgate, dup, gate_weight, up_weight, dx, workspace}), FLA_E_ALIGNMENT);
  if (M == 0) return FLA_OK;
  const TilePlan plan = plan_dx(M, F, K);
  FLA_REQUIRE(plan.splits == 1 || workspace, FLA_E_INVALID);
  GradParams p{};
  p.dg = (const char*)dgate, p.du = (const char*)dup, p.a = (const char*)gate_weight, p.b = (const char*)up_weight, p.y = dx, p.part = workspace;
  p.M = M, p.F = F, p.K = K, p.ld = ld, p.splits = plan.splits;
  hipStream_t st = (hipStream_t)stream;
  return dtype == FLA_BF16 ? launch_dx<bf16>(p, plan.kind, st) : launch_dx<f16>(p, plan.kind, st);
}

extern "C" int fla_gated_linear_bwd_dw_splits(int64_t M, int64_t F, int64_t K, int both) {
  return M <= 0 || F <= 0 || K <= 0 ? 1 : plan_dw(M, F, K, both ? 2 : 1).splits;
}

extern "C" int fla_gated_linear_bwd_dw(const void* dgate, const void* dup, const void* x, void* dgate_weight, void* dup_weight, int64_t ld, int64_t M,
                                       int64_t F, int64_t K, int dtype, float* workspace, fla_stream_t stream) {
  FLA_REQUIRE(x && (dgate_weight || dup_weight) && (!dgate_weight || dgate) && (!dup_weight || dup) && M > 0 && F > 0 && K > 0, FLA_E_INVALID);
  FLA_REQUIRE(dtype == FLA_BF16 || dtype == FLA_F16, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(sizes_ok(M, F, K) && K % 8 == 0 && ld >= F && ld % 8 == 0 && ld < F + 8, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(aligned16({dgate, dup, x, dgate_weight, dup_weight, workspace}), FLA_E_ALIGNMENT);
  const TilePlan plan = plan_dw(M, F, K, dgate_weight && dup_weight ? 2 : 1);
  FLA_REQUIRE(plan.splits == 1 || workspace, FLA_E_INVALID);
  GradParams p{};
  p.dg = (const char*)dgate, p.du = (const char*)dup, p.a = (const char*)x, p.y = dgate_weight, p.y2 = dup_weight, p.part = workspace;
  p.M = M, p.F = F, p.K = K, p.ld = ld, p.splits = plan.splits;
  hipStream_t st = (hipStream_t)stream;
  return dtype == FLA_BF16 ? launch_dw<bf16>(p, plan.kind, st) : launch_dw<f16>(p, plan.kind, st);
}
