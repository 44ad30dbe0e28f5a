// Product of rows in 8-bit integers with the epilogue of a projection:
//   y[m,n] = act(sx[m] sw[n] sum_k x[m,k] w[n,k] + bias[n]) + residual[m,n],   a scale per row of x (token) and of w (channel), act: none, silu, gelu, relu
// Sums are exact in 32 bits: K is at most 131056, where 128 * 128 * K is still below 2^31.  They are rounded to fp32 once (2^-24), and scaled, activated and
// added to the residual there; results leave in 16 bits or in fp32.  The tiles of matrix_tiles.h and, up to 64 rows of x, the panels of matrix_panels.h.
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
  bool wide;                // rows of y can be written 16 bytes at a time
};

// Four consecutive n of row m (of which those below N exist) from their sums
template <typename O, int ACT>
FLA_DEVICE void int8_values(const Int8Params& p, int64_t m, int64_t n, i32x4 sums, float sx, f32x4 sw, f32x4 bias, float* v) {
  // (erff for fp32 results; the published formula, 1.5e-7, is far below a step of 16 bits)
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const float t = fmaf((float)sums[r], sx * sw[r], bias[r]);
    v[r] = sizeof(O) == 2 ? activate_gate<ACT>(t) : activate<ACT>(t);
  }
  if (p.res && m < p.M) {
    float r[4] = {0.f, 0.f, 0.f, 0.f};
    const int64_t at = m * p.N + n;
    if (n + 4 <= p.N) {
      if (p.res_f32) load_some<float, 4, true>((const float*)p.res + at, 4, r);
      else load_some<O, 4, true>((const O*)p.res + at, 4, r);
    } else {
#pragma unroll 1
      for (int i = (int)(p.N - n) - 1; i >= 0; --i) {
        r[3] = r[2], r[2] = r[1], r[1] = r[0];
        r[0] = p.res_f32 ? ((const float*)p.res)[at + i] : (float)((const O*)p.res)[at + i];
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += r[i];
  }
}
template <typename O>
FLA_DEVICE void int8_store4(const Int8Params& p, int64_t m, int64_t n, const float* v) {
  if (m >= p.M) return;
  O* y = (O*)p.y + m * p.N + n;
  if (p.wide && n + 4 <= p.N) {
    typedef O V4 __attribute__((ext_vector_type(4)));
    *(V4*)y = V4{(O)v[0], (O)v[1], (O)v[2], (O)v[3]};
  } else {
    f32x4 t = {v[0], v[1], v[2], v[3]};
    const int count = p.N - n < 4 ? (int)(p.N - n) : 4;
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

template <typename O, int BM, int BN, bool HALVES>
struct Int8Job {
  static constexpr bool kHalves = HALVES;
  typedef MatTile<int8_t, BM, BN, 2, false, false> Whole;
  typedef MatTile<int8_t, BM, HALVES ? BN / 2 : BN, 2, false, false> Half;
  static constexpr int LATER = Whole::MT * Whole::NT * 2;   // stores of 16-bit results
  static constexpr int kLds = Whole::kLds + 2 * 2 * BN * 4;

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
  // Biases and scales of the columns, two waves each, as they lie in memory; zeros where there are none
  FLA_DEVICE char* column(int side, int which) const { return lds + Whole::kLds + (side * 2 + which) * BN * 4; }
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
  }
  FLA_DEVICE f32x4 bias4(int side, int n) const {
    const char* c = column(side, 0);
    if (p.bias_f32) return *(const f32x4*)(c + n * 4);
    typedef O V4 __attribute__((ext_vector_type(4)));
    const V4 v = *(const V4*)(c + n * sizeof(O));
    return f32x4{(float)v[0], (float)v[1], (float)v[2], (float)v[3]};
  }
  // true: every store was made, 16 bytes each, and nothing was loaded
  template <typename Tile>
  FLA_DEVICE bool finish(const Tile& t, const typename Tile::acc_t (&acc)[Tile::MT][Tile::NT], int side) const {
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
      return false;
    }
    with_activation(p.act, [&](auto act) {
#pragma unroll
      for (int i = 0; i < Tile::MT; ++i) {
        const int64_t m = m0 + (t.wm * Tile::MT + i) * 32 + lr;
        const float sx = m < p.M ? p.sx[m] : 0.f;
#pragma unroll
        for (int j = 0; j < Tile::NT; ++j) {
          const i32x16 a = mat_sums<Tile>(acc, i, j);
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const int nl = (t.wn * Tile::NT + j) * 32 + 16 * q + 4 * lh;     // of the first run of four; the second is eight further
            float v[2][4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const i32x4 sums = {a[8 * q + 4 * e], a[8 * q + 4 * e + 1], a[8 * q + 4 * e + 2], a[8 * q + 4 * e + 3]};
              int8_values<O, decltype(act)::value>(p, m, n0 + nl + 8 * e, sums, sx, *(const f32x4*)(column(side, 1) + (nl + 8 * e) * 4), bias4(side, nl + 8 * e), v[e]);
            }
            if constexpr (sizeof(O) == 2) {
              const i32x4 o = mat_join(pack4<O>(v[0]), pack4<O>(v[1]));
              if (m < p.M) store_piece((O*)p.y + m * p.N, n0 + nl - 4 * lh + 8 * lh, p.N, p.wide, o);
            } else {
              int8_store4<O>(p, m, n0 + nl, v[0]);
              int8_store4<O>(p, m, n0 + nl + 8, v[1]);
            }
            mat_piece_end();
          }
        }
      }
    });
    return false;
  }
};

template <typename O, int BM, int BN, int PER_SIMD, bool HALVES>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(PER_SIMD, PER_SIMD))) void int8_tile_kernel(Int8Params p, MatGrid grid) {
  typedef Int8Job<O, BM, BN, HALVES> Job;
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
    with_activation(p.act, [&](auto act) { int8_values<O, decltype(act)::value>(p, m, n, sums[0], m < p.M ? p.sx[m] : 0.f, sw, bias, v); });
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
  with_activation(p.act, [&](auto act) { int8_values<O, decltype(act)::value>(p, m, n, sums, p.sx[m], sw, bias, v); });
  int8_store4<O>(p, m, n, v);
}

constexpr int64_t kPanelRows = 64;   // of x; more go to the tiles
TilePlan plan_int8(int64_t M, int64_t N, int64_t K) { return plan_tiles(M, N, fla_cdiv(K, kSliceBytes), 1); }

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
  const TilePlan plan = plan_int8(p.M, p.N, p.K);
  FLA_REQUIRE(plan.splits == 1 || p.part, FLA_E_INVALID);
  p.splits = plan.splits;
  MatGrid g{};
  dim3 grid;
  const int rc = grid_of(plan.kind, fla_cdiv(p.M, kTileM[plan.kind]), fla_cdiv(p.N, kTileN[plan.kind]), p.splits, &g, &grid);
  if (rc != FLA_OK) return rc;
  if (plan.kind == kBig) hipLaunchKernelGGL((int8_tile_kernel<O, 256, 256, 1, true>), grid, dim3(256), 0, st, p, g);
  else if (plan.kind == kMiddle) hipLaunchKernelGGL((int8_tile_kernel<O, 128, 128, 2, false>), grid, dim3(256), 0, st, p, g);
  else hipLaunchKernelGGL((int8_tile_kernel<O, 64, 128, 3, false>), grid, dim3(256), 0, st, p, g);
  FLA_CHECK_LAUNCH();
  if (p.splits > 1) {
    hipLaunchKernelGGL((int8_finish_kernel<O>), dim3((unsigned)fla_cdiv(p.M * fla_cdiv(p.N, 4), 256)), dim3(256), 0, st, p);
    FLA_CHECK_LAUNCH();
  }
  return FLA_OK;
}

}  // namespace

extern "C" int fla_int8_linear_splits(int64_t M, int64_t N, int64_t K) {
  return M <= kPanelRows || N <= 0 || K <= 0 ? 1 : plan_int8(M, N, K).splits;
}

extern "C" int fla_int8_linear(const void* x, const float* x_scale, const void* weight, const float* weight_scale, const void* bias,
                               int bias_dtype, const void* residual, int residual_dtype, void* y, int64_t M, int64_t N, int64_t K,
                               int activation, int dtype, void* workspace, fla_stream_t stream) {
  FLA_REQUIRE(x && x_scale && weight && weight_scale && y && M >= 0 && N > 0 && K > 0, FLA_E_INVALID);
  FLA_REQUIRE(activation >= FLA_ACT_NONE && activation <= FLA_ACT_RELU, FLA_E_INVALID);
  FLA_REQUIRE(dtype == FLA_BF16 || dtype == FLA_F16 || dtype == FLA_F32, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(!bias || bias_dtype == dtype || bias_dtype == FLA_F32, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(!residual || residual_dtype == dtype || residual_dtype == FLA_F32, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(sizes_ok(M, N, K) && K % 16 == 0 && K <= FLA_INT8_MAX_K, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(aligned16({x, weight, workspace}) && aligned4({bias}), FLA_E_ALIGNMENT);
  if (M == 0) return FLA_OK;
  Int8Params p{};
  p.x = (const char*)x, p.w = (const char*)weight, p.sx = x_scale, p.sw = weight_scale, p.bias = bias, p.res = residual, p.y = y;
  p.part = (int*)workspace, p.M = M, p.N = N, p.K = K, p.act = activation, p.splits = 1;
  p.bias_f32 = bias_dtype == FLA_F32, p.res_f32 = residual_dtype == FLA_F32, p.wide = N % 8 == 0 && aligned16({y});
  hipStream_t st = (hipStream_t)stream;
  return dtype == FLA_BF16 ? launch_int8<bf16>(p, st) : dtype == FLA_F16 ? launch_int8<f16>(p, st) : launch_int8<float>(p, st);
}
