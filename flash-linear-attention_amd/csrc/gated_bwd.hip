// Gradients of the gated product  h = act(g) u,  g = x Wg' + bg,  u = x Wu' + bu:
//   dg = dh u act'(g),   du = dh act(g),   dx = dg Wg + du Wu,   dWg = dg' x,   dWu = du' x,   dbg, dbu: column sums of dg and du
// dg and du in one pass over dh, g and u (HBM-bound), with the column sums of the biases' gradients; dx as one product over both halves of the
// contraction (no rounding between them), its second operand strided in memory; the weights' gradients as one launch of products with both operands strided.
#include "linear_epilogue.h"
#include "matrix_plan.h"
#include "matrix_tiles.h"
#include "row_vec.h"

namespace {

struct GatedBwdParams {
  const void* dh;             // [M,F]
  const float *g, *u;         // [M,ld]
  void *dg, *du;              // [M,ld]: columns behind F are zeros
  float *pg, *pu;             // partial sums [gridDim.y, F], rows pld apart, or NULL
  int64_t M, F, ld, pld, rows;     // rows: of a workgroup
  int act;
};

// HBM-bound: 8192 x 5632 in 152 - 156 us, 4.1 - 4.2 TB/s of dh, g, u, dg and du (646 MB, of them 369 for g and u in fp32; a large copy reaches 5.1; four columns a thread, whole kilobytes a wave, was no faster).  dg and du leave in the operands' type, since the matrix instructions take
// nothing wider: half a step each.  The biases' gradients are sums of what was not rounded.
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
        Row8<float>::load(p.g + m * p.ld + col, g);
        Row8<float>::load(p.u + m * p.ld + col, u);
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
    if (part && n < p.F) part[blockIdx.y * p.pld + n] = ((sum[which][0][c] + sum[which][1][c]) + sum[which][2][c]) + sum[which][3][c];
  }
}

struct GradParams {
  const char *dg, *du;       // [M,ld]
  const char *a, *b;         // dx: Wg, Wu [F,K];  weights' gradients: x [M,K], -
  void *y, *y2;              // dx [M,K];  dWg, dWu [F,K], either may be NULL
  float* part;               // sums of slices [splits, (2,) rows, K], or NULL
  int64_t M, F, K, ld;       // K: columns of the operands, a multiple of 8
  int64_t columns;           // of the results, those below K that are wanted
  int splits;
};

// A tile of a gradient of `rows` rows of `columns` elements, or of its sums of K; 1: every store was made, 16 bytes each
template <typename T, typename Tile>
FLA_DEVICE int grad_store(const Tile& t, const typename Tile::acc_t (&acc)[Tile::MT][Tile::NT], T* y, float* part, int64_t m0, int64_t n0, int64_t rows, int64_t K, int64_t columns) {
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
          if (m < rows) store_piece(y + m * columns, n + 16 * q + 8 * lh, columns, o);
        }
      }
      mat_piece_end();
    }
  }
  return !part && m0 + Tile::MT * 64 <= rows && n0 + Tile::NT * 64 <= columns;
}

// 8192 x 2048 from 2 x 5632: 304 - 326 us, 1.2 PFLOP/s, one tile for each CU: 2 x 88 slices at 1.8 us, first copies and stores included.
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
  FLA_DEVICE int finish(const Tile& t, const typename Tile::acc_t (&acc)[Tile::MT][Tile::NT], int) const {
    return grad_store(t, acc, (T*)p.y, p.splits > 1 ? p.part + blockIdx.y * p.M * p.K : nullptr, m0, n0, p.M, p.K, p.columns);
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

// 2 x 5632 x 2048 from 8192 rows: 325 - 349 us; 352 tiles for 256 CUs, of which 96 go as half tiles (as 352 workgroups of a tile each: 371 - 379).
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
  FLA_DEVICE int finish(const Tile& t, const typename Tile::acc_t (&acc)[Tile::MT][Tile::NT], int) const {
    const bool second = up && p.y;
    return grad_store(t, acc, (T*)(up ? p.y2 : p.y), p.splits > 1 ? p.part + ((second ? p.splits : 0) + (int64_t)blockIdx.y) * p.F * p.K : nullptr, m0, n0, p.F, p.K, p.columns);
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

// the sums of slices [splits, rows, K], added in their order: four elements a thread, of which those in `columns` leave
template <typename T>
__global__ __launch_bounds__(256) void grad_finish_kernel(const float* part, T* y, T* y2, int64_t rows, int64_t K, int64_t columns, int splits) {
  const int64_t n = rows * K, at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= n) return;
  const float* from = part + (int64_t)blockIdx.y * splits * n + at;
  f32x4 v = *(const f32x4*)from;
  for (int s = 1; s < splits; ++s) v += *(const f32x4*)(from + s * n);
  typename Elem<T>::v4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = (T)v[i];
  T* out = blockIdx.y || !y ? y2 : y;
  if (columns == K) {
    *(typename Elem<T>::v4*)(out + at) = o;
  } else {
    const int64_t m = at / K, c = at - m * K;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + i < columns) out[m * columns + c + i] = o[i];
  }
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
    hipLaunchKernelGGL((grad_finish_kernel<T>), dim3((unsigned)fla_cdiv(n, 1024)), dim3(256), 0, st, p.part, (T*)p.y, (T*)p.y, p.M, p.K, p.columns, p.splits);
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
    hipLaunchKernelGGL((grad_finish_kernel<T>), dim3((unsigned)fla_cdiv(n, 1024), batch), dim3(256), 0, st, p.part, (T*)p.y, (T*)p.y2, p.F, p.K, p.columns, p.splits);
    FLA_CHECK_LAUNCH();
  }
  return FLA_OK;
}

}  // namespace

extern "C" int fla_gated_linear_bwd_rows(int64_t M) { return M <= 0 ? 1 : (int)(fla_cdiv(M, 256) < 32 ? 32 : fla_cdiv(M, 256)); }

extern "C" int fla_gated_linear_bwd_gate(const void* dh, const float* gate, const float* up, void* dgate, void* dup, float* dgate_bias_partial,
                                         float* dup_bias_partial, int64_t partial_ld, int64_t ld, int64_t M, int64_t F, int activation, int dtype,
                                         fla_stream_t stream) {
  FLA_REQUIRE(dh && gate && up && dgate && dup && M >= 0 && F > 0, FLA_E_INVALID);
  FLA_REQUIRE(activation >= FLA_ACT_NONE && activation <= FLA_ACT_RELU, FLA_E_INVALID);
  FLA_REQUIRE(dtype == FLA_BF16 || dtype == FLA_F16, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(sizes_ok(M, F, 1) && ld >= F && ld % 8 == 0 && ld < F + 8, FLA_E_UNSUPPORTED);
  FLA_REQUIRE((!dgate_bias_partial && !dup_bias_partial) || partial_ld >= F, FLA_E_INVALID);
  FLA_REQUIRE(aligned16({gate, up, dgate, dup}), FLA_E_ALIGNMENT);
  if (M == 0) return FLA_OK;
  GatedBwdParams p{};
  p.dh = dh, p.g = gate, p.u = up, p.dg = dgate, p.du = dup, p.pg = dgate_bias_partial, p.pu = dup_bias_partial, p.M = M, p.F = F, p.ld = ld, p.pld = partial_ld;
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
                                       int64_t columns, int64_t M, int64_t F, int64_t K, int dtype, float* workspace, fla_stream_t stream) {
  FLA_REQUIRE(dgate && dup && gate_weight && up_weight && dx && M >= 0 && F > 0 && K > 0, FLA_E_INVALID);
  FLA_REQUIRE(dtype == FLA_BF16 || dtype == FLA_F16, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(sizes_ok(M, F, K) && K % 8 == 0 && ld >= F && ld % 8 == 0 && ld < F + 8 && columns > 0 && columns <= K, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(aligned16({dgate, dup, gate_weight, up_weight, columns == K ? dx : nullptr, workspace}), FLA_E_ALIGNMENT);
  if (M == 0) return FLA_OK;
  const TilePlan plan = plan_dx(M, F, K);
  FLA_REQUIRE(plan.splits == 1 || workspace, FLA_E_INVALID);
  GradParams p{};
  p.dg = (const char*)dgate, p.du = (const char*)dup, p.a = (const char*)gate_weight, p.b = (const char*)up_weight, p.y = dx, p.part = workspace;
  p.M = M, p.F = F, p.K = K, p.ld = ld, p.columns = columns, p.splits = plan.splits;
  hipStream_t st = (hipStream_t)stream;
  return dtype == FLA_BF16 ? launch_dx<bf16>(p, plan.kind, st) : launch_dx<f16>(p, plan.kind, st);
}

extern "C" int fla_gated_linear_bwd_dw_splits(int64_t M, int64_t F, int64_t K, int both) {
  return M <= 0 || F <= 0 || K <= 0 ? 1 : plan_dw(M, F, K, both ? 2 : 1).splits;
}

extern "C" int fla_gated_linear_bwd_dw(const void* dgate, const void* dup, const void* x, void* dgate_weight, void* dup_weight, int64_t ld,
                                       int64_t columns, int64_t M, int64_t F, int64_t K, int dtype, float* workspace, fla_stream_t stream) {
  FLA_REQUIRE(x && (dgate_weight || dup_weight) && (!dgate_weight || dgate) && (!dup_weight || dup) && M > 0 && F > 0 && K > 0, FLA_E_INVALID);
  FLA_REQUIRE(dtype == FLA_BF16 || dtype == FLA_F16, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(sizes_ok(M, F, K) && K % 8 == 0 && ld >= F && ld % 8 == 0 && ld < F + 8 && columns > 0 && columns <= K, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(aligned16({dgate, dup, x, columns == K ? dgate_weight : nullptr, columns == K ? dup_weight : nullptr, workspace}), FLA_E_ALIGNMENT);
  const TilePlan plan = plan_dw(M, F, K, dgate_weight && dup_weight ? 2 : 1);
  FLA_REQUIRE(plan.splits == 1 || workspace, FLA_E_INVALID);
  GradParams p{};
  p.dg = (const char*)dgate, p.du = (const char*)dup, p.a = (const char*)x, p.y = dgate_weight, p.y2 = dup_weight, p.part = workspace;
  p.M = M, p.F = F, p.K = K, p.ld = ld, p.columns = columns, p.splits = plan.splits;
  hipStream_t st = (hipStream_t)stream;
  return dtype == FLA_BF16 ? launch_dw<bf16>(p, plan.kind, st) : launch_dw<f16>(p, plan.kind, st);
}
