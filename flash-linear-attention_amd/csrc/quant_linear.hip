// Product of 8-bit rows with the epilogue of a projection:
//   y[m,n] = act(sx[m] sw[n] sum_k x[m,k] w[n,k] + bias[n]) + residual[m,n],   x, w in e4m3, a scale per row, act: none, silu, gelu, relu
// Both operands have their contraction index contiguous.  Sums run on the 16x16x128 matrix instruction, whose order over k is the same
// permutation for both operands, so a lane takes 32 bytes of its row wherever they lie.  Rows of w are the instruction's first operand:
// a lane then holds consecutive n of one m, and writes them as one piece.
//
// Numerics.  The instruction aligns eight products (consecutive k) to the largest of them and cuts each, towards zero, at 2^-13 of the
// largest one's power of two; the sums of eight are added in fp32 (found with two products in one group and in two).  Against fp64, random
// operands give a relative error of 1.2e-5 (K = 256 .. 8192; the 16x16x32 form likewise), 1/40 of half a step of fp16, and the operands'
// own rounding to 8 bits is a thousand times that.  Results leave in 16 bits only.  The alternative, conversion to bf16 and the instruction
// that keeps whole products, runs at half the rate.
#include "fla_common.h"

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

struct LinearParams {
  const uint8_t* x;      // [M,K]
  const float* sx;       // [M]
  const uint8_t* w;      // [N,K]
  const float* sw;       // [N]
  const void* bias;      // [N] or NULL
  const void* res;       // [M,N] or NULL
  void* y;               // [M,N]
  float* part;           // [splits, M, N]: sums of a slice of K, or NULL
  int64_t M, N, K;
  int bias_f32, res_f32, act, splits;
  bool wide;             // rows of y and of the residual can be taken 16 bytes at a time
};

template <int ACT>
FLA_DEVICE float activate(float v) {
  if (ACT == FLA_ACT_SILU) return v * __builtin_amdgcn_rcpf(1.f + __expf(-v));
  if (ACT == FLA_ACT_GELU) return 0.5f * v * (1.f + erff(v * 0.70710678f));
  if (ACT == FLA_ACT_RELU) return v < 0.f ? 0.f : v;      // (NaN stays)
  return v;
}

// both e4m3, no block scales
FLA_DEVICE f32x4 mfma8(i32x8 a, i32x8 b, f32x4 c) { return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0); }

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

// COUNT (4 or 8) consecutive n of row m from their sums.  FULL: all of them exist, and they can be taken 16 bytes at a time.
template <typename T, int COUNT, int ACT, bool FULL>
FLA_DEVICE void finish(const LinearParams& p, int64_t m, int64_t n, const float* acc, float sx, const float* sw, const float* bias) {
  const int valid = FULL || p.N - n > COUNT ? COUNT : (int)(p.N - n);
  if (m >= p.M || (!FULL && valid <= 0)) return;
  float v[COUNT], r[COUNT];
  const int64_t at = m * p.N + n;
  if (p.res) {
    if (p.res_f32) load_some<float, COUNT, FULL>((const float*)p.res + at, valid, r);
    else load_some<T, COUNT, FULL>((const T*)p.res + at, valid, r);
  }
#pragma unroll
  for (int i = 0; i < COUNT; ++i) v[i] = activate<ACT>(fmaf(acc[i], sx * sw[i], bias[i]));
  if (p.res)
#pragma unroll
    for (int i = 0; i < COUNT; ++i) v[i] += r[i];
  T* y = (T*)p.y + at;
  if (FULL) {
    typedef T vec __attribute__((ext_vector_type(COUNT)));
    vec o;
#pragma unroll
    for (int i = 0; i < COUNT; ++i) o[i] = (T)v[i];
    *(vec*)y = o;
  } else {
#pragma unroll
    for (int i = 0; i < COUNT; ++i)
      if (i < valid) y[i] = (T)v[i];
  }
}
template <typename T>
FLA_DEVICE float bias_of(const LinearParams& p, int64_t n) {
  return !p.bias || n >= p.N ? 0.f : p.bias_f32 ? ((const float*)p.bias)[n] : (float)((const T*)p.bias)[n];
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

// ------------------------------------------------------------------------------------------------ tiles
__device__ const i32x4 kZeros = {0, 0, 0, 0};

// A BM x BN tile of y for WM x WN waves.  Slices of 128 bytes of K go through LDS, RING of them: one is read while the next arrive
// straight from memory (a wave's copy instruction fills 1024 bytes: eight rows of 128).  The 16-byte pieces of a row are permuted within it by a key
// of the row: a b128 read serves lanes 0-3, 12-15, 20-27 together, then 4-11, 16-19, 28-31, and the same of the upper half (found by timing
// patterns), and with these keys each sixteen meet all 64 banks once.
template <typename T, int BM, int BN, int WM, int WN, int PER_SIMD, int RING>
__global__ __launch_bounds__(WM * WN * 64) __attribute__((amdgpu_waves_per_eu(PER_SIMD))) void linear_tile_kernel(LinearParams p) {
  constexpr int WAVES = WM * WN, BK = 128;
  constexpr int MT = BM / WM / 16, NT = BN / WN / 16;          // 16 x 16 tiles of a wave
  constexpr int CX = BM / 8 / WAVES, CW = BN / 8 / WAVES;      // copy instructions of a wave for a slice
  static_assert(NT % 2 == 0 && CX >= 1 && CW >= 1 && BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0, "whole copies");
  // (One array: the compiler tells apart the members of several, and then waits for copies in flight ahead of every read.)
  constexpr int SLICE = (BM + BN) * BK;
  __shared__ __attribute__((aligned(16))) uint8_t lds[RING * SLICE + (BM + 2 * BN) * 4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN, lr = lane & 15, lq = lane >> 4;

  // Neighbouring workgroup numbers go to different XCDs: each XCD takes a run of tiles, eight rows of tiles deep, that share operands in its L2
  const uint32_t tm_all = (uint32_t)((p.M + BM - 1) / BM), tn_all = (uint32_t)((p.N + BN - 1) / BN), total = tm_all * tn_all;
  const uint32_t xcd = blockIdx.x % 8, per = total / 8, rest = total % 8;
  const uint32_t id = xcd * per + (xcd < rest ? xcd : rest) + blockIdx.x / 8;
  const uint32_t deep = tm_all < 8 ? tm_all : 8, band = id / (deep * tn_all), in = id - band * deep * tn_all;
  const uint32_t rows_in = tm_all - band * deep < deep ? tm_all - band * deep : deep, col = in / rows_in;
  const int64_t m0 = (int64_t)(band * deep + in - col * rows_in) * BM, n0 = (int64_t)col * BN;

  // slices of K for this workgroup
  const int per_split = (int)((p.K + BK - 1) / BK + p.splits - 1) / p.splits * BK;
  const int k_first = blockIdx.y * per_split, k_end = p.K - k_first < per_split ? (int)p.K : k_first + per_split;

  // what the epilogue multiplies and adds, out of memory's latency by then
  float *sxs = (float*)(lds + RING * SLICE), *sws = sxs + BM, *bs = sws + BN;
  for (int i = tid; i < BM; i += WAVES * 64) sxs[i] = m0 + i < p.M ? p.sx[m0 + i] : 0.f;
  for (int i = tid; i < BN; i += WAVES * 64) {
    sws[i] = n0 + i < p.N ? p.sw[n0 + i] : 0.f;
    bs[i] = bias_of<T>(p, n0 + i);
  }

  // what this lane copies: piece `lane % 8` of LDS row r holds piece (lane % 8) ^ key(r) of the matrix row
  auto w_key = [](int r) { return (r & 3) | (r >> 3 & 1) << 2; };
  const uint8_t *xb = p.x + m0 * p.K, *wb = p.w + n0 * p.K;
  const int K = (int)p.K, rows_m = p.M - m0 < BM ? (int)(p.M - m0) : BM, rows_n = p.N - n0 < BN ? (int)(p.N - n0) : BN;
  uint32_t at[CX + CW];
#pragma unroll
  for (int q = 0; q < CX; ++q) {
    const int r = (wave * CX + q) * 8 + lane / 8;
    at[q] = (uint32_t)(r < rows_m ? r : rows_m - 1) * K + ((lane & 7) ^ (r & 7)) * 16;
  }
#pragma unroll
  for (int q = 0; q < CW; ++q) {
    const int r = (wave * CW + q) * 8 + lane / 8;
    at[CX + q] = (uint32_t)(r < rows_n ? r : rows_n - 1) * K + ((lane & 7) ^ w_key(r)) * 16;
  }
  auto copy = [&](int k0, int buf) {
#pragma unroll
    for (int q = 0; q < CX + CW; ++q) {
      const int row = q < CX ? (wave * CX + q) * 8 : BM + (wave * CW + q - CX) * 8;
      const uint8_t* from = (q < CX ? xb : wb) + k0 + at[q];
      if (k0 + BK > K) {   // (uniform) beyond the end of K, in multiples of 16: zeros
        const int piece = ((lane & 7) ^ (q < CX ? row + lane / 8 & 7 : w_key(row - BM + lane / 8))) * 16;
        if (k0 + piece >= K) from = (const uint8_t*)&kZeros;
      }
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                       (__attribute__((address_space(3))) void*)(lds + buf * SLICE + row * BK), 16, 0, 0);
    }
  };

  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  // 32 bytes of a row's slice: pieces lq and lq + 4
  auto fragment = [&](const uint8_t* base, int row, int key) {
    const uint8_t* r = base + row * BK;
    const i32x4 a = *(const i32x4*)(r + (lq ^ key) * 16), b = *(const i32x4*)(r + ((lq + 4) ^ key) * 16);
    return i32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  };
#pragma unroll
  for (int d = 0; d + 1 < RING; ++d)
    if (k_first + d * BK < k_end) copy(k_first + d * BK, d);
  int buf = 0;
  for (int k0 = k_first; k0 < k_end; k0 += BK, buf = buf + 1 < RING ? buf + 1 : 0) {
    // this wave's part of the slice has arrived (copies arrive in order, those of RING - 2 slices may follow)
    if (RING > 2 && k0 + (RING - 2) * BK < k_end) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"i"((RING - 2) * (CX + CW)) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();                                 // everybody's has, and the slice before is no longer read
    if (k0 + (RING - 1) * BK < k_end) copy(k0 + (RING - 1) * BK, buf ? buf - 1 : RING - 1);
    const uint8_t *xs = lds + buf * SLICE, *ws = xs + BM * BK;
    i32x8 wf[NT], xf[MT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      // Lane row lr of tile j is row 32 (j / 2) + 8 (lr / 4) + 4 (j % 2) + lr % 4 of the wave's: a lane's sums of two tiles are eight
      // consecutive n, and those of the four lanes of a row 32.
      const int r = wn * NT * 16 + (j >> 1) * 32 + (lr >> 2) * 8 + (j & 1) * 4 + (lr & 3);
      wf[j] = fragment(ws, r, w_key(r));
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int r = (wm * MT + i) * 16 + lr;
      xf[i] = fragment(xs, r, r & 7);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] = mfma8(wf[j], xf[i], acc[i][j]);
    // a row of products while the next one's operand is read
    __builtin_amdgcn_sched_group_barrier(0x100, 2 * NT + 2, 0);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      if (i + 1 < MT) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, NT, 0);
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // no copy into LDS outlives the workgroup
  const int lm = wm * MT * 16 + lr, ln = wn * NT * 16 + lq * 8;
  if (p.splits > 1) {   // linear_finish_kernel adds the slices' sums
    float* part = p.part + blockIdx.y * p.M * p.N;
#pragma unroll
    for (int h = 0; h < NT / 2; ++h)
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int64_t m = m0 + lm + i * 16, n = n0 + ln + h * 32;
        if (m >= p.M) continue;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          float* to = part + m * p.N + n + 4 * q;
          const f32x4 v = acc[i][2 * h + q];
          if (n + 4 * q + 4 <= p.N) {
            *(f32x4_any*)to = v;
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (n + 4 * q + r < p.N) to[r] = v[r];
          }
        }
      }
    return;
  }
  auto epilogue = [&](auto act, auto full) {
    float sx[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) sx[i] = sxs[lm + i * 16];
#pragma unroll
    for (int h = 0; h < NT / 2; ++h) {
      float sw[8], bias[8];
      load_some<float, 8, true>(sws + ln + h * 32, 8, sw);
      load_some<float, 8, true>(bs + ln + h * 32, 8, bias);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        float v[8];
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = acc[i][2 * h][r], v[4 + r] = acc[i][2 * h + 1][r];
        finish<T, 8, decltype(act)::value, decltype(full)::value>(p, m0 + lm + i * 16, n0 + ln + h * 32, v, sx[i], sw, bias);
      }
    }
  };
  with_activation(p.act, [&](auto act) {
    if (p.wide && n0 + BN <= p.N) epilogue(act, Const<true>());
    else epilogue(act, Const<false>());
  });
}

// ------------------------------------------------------------------------------------------------ few rows
// At most MT x 16 rows of x against 16 rows of w: the bytes of w bound it, and those of x out of L2 from 32 rows on.  The waves take slices of 128 bytes
// of K in turn, each through RING pieces of LDS of its own, waiting for nobody until the sums are added.  (Operands loaded straight into the instruction's
// registers meet 16 rows with every 16 lanes and pass 17 bytes a clock and CU, whole 128-byte pieces 50: 48 x 2048 x 8192 took 16.6 us, with copies 8.3, w in the
// last-level cache; out of HBM 11.2.)
template <typename T, int MT, int WAVES, int RING>
__global__ __launch_bounds__(WAVES * 64) void linear_panel_kernel(LinearParams p) {
  constexpr int BK = 128, ROWS = (MT + 1) * 16, COPIES = ROWS / 8;   // rows of x, then those of w
  __shared__ __attribute__((aligned(16))) uint8_t lds[WAVES * RING * ROWS * BK];
  static_assert(sizeof(lds) >= WAVES * MT * 64 * 16, "the sums take the place of the slices");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 15, lq = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const uint8_t* wb = p.w + n0 * p.K;
  const int K = (int)p.K, rows_n = p.N - n0 < 16 ? (int)(p.N - n0) : 16, rows_m = (int)p.M, piece = ((lane & 7) ^ (lane >> 3)) * 16;
  uint32_t at[COPIES];
#pragma unroll
  for (int q = 0; q < COPIES; ++q) {
    const int r = (q < 2 * MT ? q : q - 2 * MT) * 8 + lane / 8, rows = q < 2 * MT ? rows_m : rows_n;
    at[q] = (uint32_t)(r < rows ? r : rows - 1) * K + piece;
  }
  uint8_t* mine = lds + wave * RING * ROWS * BK;
  auto copy = [&](int k0, int buf) {   // slices beyond the end are zeros
#pragma unroll
    for (int q = 0; q < COPIES; ++q) {
      const uint8_t* from = (q < 2 * MT ? p.x : wb) + k0 + at[q];
      if (k0 + BK > K && k0 + piece >= K) from = (const uint8_t*)&kZeros;
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                       (__attribute__((address_space(3))) void*)(mine + (buf * ROWS + q * 8) * BK), 16, 0, 0);
    }
  };
  auto fragment = [&](int buf, int row) {   // pieces lq and lq + 4 of a row (keyed by the row, as in the tiles)
    const uint8_t* r = mine + (buf * ROWS + row) * BK;
    const i32x4 a = *(const i32x4*)(r + (lq ^ (row & 7)) * 16), b = *(const i32x4*)(r + ((lq + 4) ^ (row & 7)) * 16);
    return i32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  };
  f32x4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int d = 0; d + 1 < RING; ++d) copy((wave + d * WAVES) * BK, d);
  int buf = 0;
  for (int k0 = wave * BK; k0 < K; k0 += WAVES * BK) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the slice that the next copy replaces has been read
    copy(k0 + (RING - 1) * WAVES * BK, buf ? buf - 1 : RING - 1);
    asm volatile("s_waitcnt vmcnt(%0)" ::"i"((RING - 1) * COPIES) : "memory");   // (loads arrive in order: this slice has)
    const i32x8 wf = fragment(buf, MT * 16 + lr);
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i] = mfma8(wf, fragment(buf, i * 16 + lr), acc[i]);
    buf = buf + 1 < RING ? buf + 1 : 0;
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __syncthreads();
  f32x4(*sums)[MT][64] = (f32x4(*)[MT][64])lds;
#pragma unroll
  for (int i = 0; i < MT; ++i) sums[wave][i][lane] = acc[i];
  __syncthreads();
  for (int i = wave; i < MT; i += WAVES) {
    f32x4 t = sums[0][i][lane];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) t += sums[w][i][lane];
    const int64_t m = i * 16 + lr, n = n0 + lq * 4;
    float v[4] = {t[0], t[1], t[2], t[3]}, sw[4], bias[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      sw[c] = n + c < p.N ? p.sw[n + c] : 0.f;
      bias[c] = bias_of<T>(p, n + c);
    }
    const float sx = m < p.M ? p.sx[m] : 0.f;
    with_activation(p.act, [&](auto act) {
      constexpr int A = decltype(act)::value;
      if (p.wide && n0 + 16 <= p.N) finish<T, 4, A, true>(p, m, n, v, sx, sw, bias);
      else finish<T, 4, A, false>(p, m, n, v, sx, sw, bias);
    });
  }
}

// y from the sums of slices of K, added in their order: four columns a thread
template <typename T>
__global__ __launch_bounds__(256) void linear_finish_kernel(LinearParams p) {
  const int64_t per = (p.N + 3) / 4, id = (int64_t)blockIdx.x * 256 + threadIdx.x, m = id / per, n = id % per * 4;
  if (m >= p.M) return;
  const int valid = p.N - n < 4 ? (int)(p.N - n) : 4;
  float v[4] = {0.f, 0.f, 0.f, 0.f}, sw[4], bias[4];
  for (int s = 0; s < p.splits; ++s) {
    const float* from = p.part + (s * p.M + m) * p.N + n;
    float t[4];
    if (valid == 4) load_some<float, 4, true>(from, 4, t);
    else load_some<float, 4, false>(from, valid, t);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += t[i];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    sw[i] = i < valid ? p.sw[n + i] : 0.f;
    bias[i] = bias_of<T>(p, n + i);
  }
  const float sx = p.sx[m];
  with_activation(p.act, [&](auto act) {
    if (p.wide) finish<T, 4, decltype(act)::value, true>(p, m, n, v, sx, sw, bias);
    else finish<T, 4, decltype(act)::value, false>(p, m, n, v, sx, sw, bias);
  });
}

template <typename T, int BM, int BN, int WM, int WN, int PER_SIMD, int RING>
int launch_tiles(const LinearParams& p, hipStream_t st) {
  const int64_t total = fla_cdiv(p.M, BM) * fla_cdiv(p.N, BN);
  FLA_REQUIRE(total < (int64_t)1 << 32 >> (WM * WN == 8 ? 9 : 8), FLA_E_UNSUPPORTED);   // (a launch is less than 2^32 threads)
  hipLaunchKernelGGL((linear_tile_kernel<T, BM, BN, WM, WN, PER_SIMD, RING>), dim3((unsigned)total, p.splits), dim3(WM * WN * 64), 0, st, p);
  FLA_CHECK_LAUNCH();
  if (p.splits > 1) {
    hipLaunchKernelGGL((linear_finish_kernel<T>), dim3((unsigned)fla_cdiv(p.M * fla_cdiv(p.N, 4), 256)), dim3(256), 0, st, p);
    FLA_CHECK_LAUNCH();
  }
  return FLA_OK;
}
// Four waves to a workgroup; eight where there are fewer workgroups than CUs (1 x 2048 x 8192: 5.5 us instead of 6.5; 16 x 50000 x 2048: 26 instead of 22).
template <typename T, int MT>
int launch_panel(const LinearParams& p, hipStream_t st) {
  const int64_t grid = fla_cdiv(p.N, 16);
  FLA_REQUIRE(grid < (int64_t)1 << 32 >> 8, FLA_E_UNSUPPORTED);   // (a launch is less than 2^32 threads)
  if (grid < 256) hipLaunchKernelGGL((linear_panel_kernel<T, MT, 8, 2>), dim3((unsigned)grid), dim3(512), 0, st, p);
  else hipLaunchKernelGGL((linear_panel_kernel<T, MT, 4, 2>), dim3((unsigned)grid), dim3(256), 0, st, p);
  FLA_CHECK_LAUNCH();
  return FLA_OK;
}
// Which kernel, and how many slices of K.  Measured (us, in a captured graph, twelve sets of w or 600 MB of them in turn; M x N x K; the floor is the
// bytes').  Twelve sets of at most 21 MB stay in the last-level cache, so w comes out of HBM in the rows with more than that only; out of HBM what
// plan_linear takes needs 4.2 for 1 x 4096 x 2048, 11.2 for 48 x 2048 x 8192, 5.1 for 48 x 2048 x 2048, 15.9 for 100 x 2048 x 8192, 16.1 for 256 x 4096 x 4096,
// 20.2 for 500 x 4096 x 4096 and 27.6 for 1000 x 4096 x 4096.
//                       floor  panels  64 x 64 in 1, 2, 4, 8 slices   128 x 64   256 x 256
//   1 x 16384 x 2048      6.5     8.7   10.1                            11.8        26
//   16 x 16384 x 2048     6.6     8.5   10.2  13.1  15                  11.9        26
//   64 x 16384 x 2048     6.9    15.3   10.5  15.2  19.5                12.5        27
//   64 x 16384 x 8192    26.5    45.7   35    38    39    46            37.6        94
//   16 x 50000 x 2048    20.1    22.0   24.5                            27.6        30
//   64 x 50000 x 2048    21.1    40.6   26.5  38.8                      32          31
//   64 x 8192 x 4096      6.7    14.8   17.0  15.9  15.3  19.1          19.7        49
//   48 x 2048 x 8192      3.4     8.3   25.1  17.4  12.5  11.7          33          91
//   48 x 2048 x 2048      0.9     4.3
//   100 x 2048 x 8192     3.5           25.2  17.9  13.5  14.5          33          92
//   200 x 16384 x 2048    7.8           21.2  34    45                  16.2        30
//   256 x 4096 x 4096     3.9           14.6  18.3  20.8  24.7          18.5        50
//   1000 x 4096 x 4096    5.6           32    43    62                  24.1        51
//   8191 x 8192 x 2048   32.5 (115 at the rate of 8192^3)               176         149 (1.84 PFLOP/s; 8192^3: 2.45)
enum LinearKind { kPanel, kTile64, kTile128x64, kTile256 };
struct LinearPlan {
  LinearKind kind;
  int splits;
};
LinearPlan plan_linear(int64_t M, int64_t N, int64_t K) {
  // tiles of 256 x 256 need the fewest bytes, tiles of 128 x 64 a quarter of the rows and columns to fill the chip
  if (M > 64 && fla_cdiv(M, 256) * fla_cdiv(N, 256) >= 192) return {kTile256, 1};
  if (M > 64 && fla_cdiv(M, 128) * fla_cdiv(N, 64) >= 256) return {kTile128x64, 1};
  // The others by an estimate in us.
  const int64_t tiles = fla_cdiv(M, 64) * fla_cdiv(N, 64), slices = fla_cdiv(K, 128);
  const double w_bytes = (double)N * (double)K;
  LinearPlan best{kTile64, 1};
  double time = 0;
  for (int splits = 1; splits <= 16; splits *= 2) {
    if (splits > 1 && (tiles * splits > 1024 || slices < 4 * splits)) break;
    // 0.43 us a slice, half of that more for every further workgroup on the CU, or w at 4.5 TB/s; the second launch 4 us, and its sums go out and in
    const double load = (double)(tiles * splits) / 256, work = 0.43 * (double)fla_cdiv(slices, splits) * (load > 1 ? 0.5 + 0.5 * load : 1);
    const double bytes = w_bytes / 4.5e6 + 0.5;
    const double t = 2.5 + (work > bytes ? work : bytes) + (splits > 1 ? 4 + 2e-6 * splits * (double)(M * N) : 0);
    if (splits == 1 || t < time) best.splits = splits, time = t;
  }
  best.splits = (int)fla_cdiv(slices, fla_cdiv(slices, best.splits));   // none of them empty
  if (M <= 64) {
    // w at 4.6 TB/s, and 16 rows of it with all of x for every workgroup: 13 TB/s out of L2, 0.1 of them to a CU
    const int64_t groups = fla_cdiv(N, 16);
    const double panel = (double)(16 + fla_cdiv(M, 16) * 16) * (double)K;
    double t = w_bytes / 4.6e6;
    if (panel * (double)groups / 13e6 > t) t = panel * (double)groups / 13e6;
    if (panel * (double)fla_cdiv(groups, 256) / 1e5 > t) t = panel * (double)fla_cdiv(groups, 256) / 1e5;
    if (3 + t < time) return {kPanel, 1};
  }
  return best;
}

template <typename T>
int launch_linear(const LinearParams& p, LinearKind kind, hipStream_t st) {
  switch (kind) {
    case kTile256: return launch_tiles<T, 256, 256, 2, 4, 2, 2>(p, st);
    case kTile128x64: return launch_tiles<T, 128, 64, 2, 2, 2, 3>(p, st);
    case kTile64: return launch_tiles<T, 64, 64, 2, 2, 3, 3>(p, st);
    default: break;
  }
  if (p.M <= 16) return launch_panel<T, 1>(p, st);
  if (p.M <= 32) return launch_panel<T, 2>(p, st);
  if (p.M <= 48) return launch_panel<T, 3>(p, st);
  return launch_panel<T, 4>(p, st);
}

}  // namespace

extern "C" int fla_quant_linear_splits(int64_t M, int64_t N, int64_t K) {
  return M <= 0 || N <= 0 || K <= 0 ? 1 : plan_linear(M, N, K).splits;
}

extern "C" int fla_quant_linear(const void* x, const float* x_scale, const void* weight, const float* weight_scale, const void* bias,
                                int bias_dtype, const void* residual, int residual_dtype, void* y, int64_t M, int64_t N, int64_t K,
                                int activation, int dtype, float* workspace, fla_stream_t stream) {
  FLA_REQUIRE(x && x_scale && weight && weight_scale && y && M >= 0 && N > 0 && K > 0, FLA_E_INVALID);
  FLA_REQUIRE(activation >= FLA_ACT_NONE && activation <= FLA_ACT_RELU, FLA_E_INVALID);
  FLA_REQUIRE(dtype == FLA_BF16 || dtype == FLA_F16, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(!bias || bias_dtype == dtype || bias_dtype == FLA_F32, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(!residual || residual_dtype == dtype || residual_dtype == FLA_F32, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(K % 16 == 0 && K <= 1 << 23 && N <= 0x7fffffff && M <= 0x7fffffff, FLA_E_UNSUPPORTED);
  FLA_REQUIRE((((uintptr_t)x) | ((uintptr_t)weight)) % 16 == 0, FLA_E_ALIGNMENT);
  if (M == 0) return FLA_OK;
  LinearParams p{};
  p.x = (const uint8_t*)x, p.sx = x_scale, p.w = (const uint8_t*)weight, p.sw = weight_scale, p.bias = bias, p.res = residual, p.y = y;
  p.M = M, p.N = N, p.K = K, p.act = activation;
  const LinearPlan plan = plan_linear(M, N, K);
  FLA_REQUIRE(plan.splits == 1 || workspace, FLA_E_INVALID);
  p.splits = plan.splits, p.part = workspace;
  p.bias_f32 = bias_dtype == FLA_F32, p.res_f32 = residual_dtype == FLA_F32;
  p.wide = N % 8 == 0 && (((uintptr_t)residual) | ((uintptr_t)y)) % 16 == 0;
  hipStream_t st = (hipStream_t)stream;
  return dtype == FLA_BF16 ? launch_linear<bf16>(p, plan.kind, st) : launch_linear<f16>(p, plan.kind, st);
}
