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

enum { kNone = FLA_ACT_NONE, kSilu = FLA_ACT_SILU, kGelu = FLA_ACT_GELU, kRelu = FLA_ACT_RELU };
FLA_DEVICE float activate(float v, int act) {
  if (act == kSilu) return v * __builtin_amdgcn_rcpf(1.f + __expf(-v));
  if (act == kGelu) return 0.5f * v * (1.f + erff(v * 0.70710678f));
  if (act == kRelu) return v < 0.f ? 0.f : v;      // (NaN stays)
  return v;
}

FLA_DEVICE f32x4 mfma8(i32x8 a, i32x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);   // both e4m3, no block scales
}

// COUNT (4, 8 or 16) consecutive n of row m from their sums
template <typename T, int COUNT>
FLA_DEVICE void finish(const LinearParams& p, int64_t m, int64_t n0, const float* acc) {
  if (m >= p.M || n0 >= p.N) return;
  const float sx = p.sx[m];
  float v[COUNT];
#pragma unroll
  for (int i = 0; i < COUNT; ++i) {
    const int64_t n = n0 + i < p.N ? n0 + i : p.N - 1;
    float t = acc[i] * (sx * p.sw[n]);
    if (p.bias) t += p.bias_f32 ? ((const float*)p.bias)[n] : (float)((const T*)p.bias)[n];
    v[i] = activate(t, p.act);
  }
  const int64_t at = m * p.N + n0;
  if (p.wide && n0 + COUNT <= p.N) {
    typedef T out_t __attribute__((ext_vector_type(COUNT < 8 ? COUNT : 8)));
    constexpr int W = COUNT < 8 ? COUNT : 8;
#pragma unroll
    for (int h = 0; h < COUNT; h += W) {
      if (p.res) {
        if (p.res_f32) {
#pragma unroll
          for (int i = 0; i < W; i += 4) {
            const f32x4 r = *(const f32x4*)((const float*)p.res + at + h + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[h + i + j] += r[j];
          }
        } else {
          const out_t r = *(const out_t*)((const T*)p.res + at + h);
#pragma unroll
          for (int i = 0; i < W; ++i) v[h + i] += (float)r[i];
        }
      }
      out_t o;
#pragma unroll
      for (int i = 0; i < W; ++i) o[i] = (T)v[h + i];
      *(out_t*)((T*)p.y + at + h) = o;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < COUNT; ++i) {
    if (n0 + i >= p.N) break;
    if (p.res) v[i] += p.res_f32 ? ((const float*)p.res)[at + i] : (float)((const T*)p.res)[at + i];
    ((T*)p.y)[at + i] = (T)v[i];
  }
}

// ------------------------------------------------------------------------------------------------ tiles
__device__ const i32x4 kZeros = {0, 0, 0, 0};

// A BM x BN tile of y for WM x WN waves; slices of 128 bytes of K go through LDS, two of them: one is read while the next arrives
// straight from memory (a wave's copy instruction fills 1024 bytes: eight rows of 128).  The 16-byte pieces of a row are permuted within it by
// a key of the row, so that eight lanes that read the same piece of eight rows meet all banks.
template <typename T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64) void linear_tile_kernel(LinearParams p) {
  constexpr int THREADS = WM * WN * 64, WAVES = WM * WN, BK = 128;
  constexpr int MT = BM / WM / 16, NT = BN / WN / 16;          // 16 x 16 tiles of a wave
  constexpr int CX = BM / 8 / WAVES, CW = BN / 8 / WAVES;      // copy instructions of a wave for a slice
  static_assert(CX >= 1 && CW >= 1 && BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0, "whole copies");
  __shared__ __attribute__((aligned(16))) uint8_t lds[2][(BM + BN) * BK];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;

  // Neighbouring workgroup numbers go to different XCDs: each XCD takes a run of tiles, eight rows of tiles deep, that share operands in its L2
  const int64_t tm_all = (p.M + BM - 1) / BM, tn_all = (p.N + BN - 1) / BN, total = tm_all * tn_all;
  const int64_t bid = blockIdx.x, xcd = bid % 8, per = total / 8, rest = total % 8;
  const int64_t id = xcd * per + (xcd < rest ? xcd : rest) + bid / 8;
  const int64_t deep = 8, band = id / (deep * tn_all), in = id % (deep * tn_all);
  const int64_t rows_in = tm_all - band * deep < deep ? tm_all - band * deep : deep;
  const int64_t m0 = (band * deep + in % rows_in) * BM, n0 = in / rows_in * BN;

  // what this lane copies: piece `lane % 8` of LDS row r holds piece (lane % 8) ^ key(r) of the matrix row
  const uint8_t* src[CX + CW];
  int piece[CX + CW];
#pragma unroll
  for (int q = 0; q < CX; ++q) {
    const int r = (wave * CX + q) * 8 + lane / 8;
    const int64_t m = m0 + r < p.M ? m0 + r : p.M - 1;
    piece[q] = ((lane & 7) ^ (r & 7)) * 16;
    src[q] = p.x + m * p.K;
  }
#pragma unroll
  for (int q = 0; q < CW; ++q) {
    const int r = (wave * CW + q) * 8 + lane / 8;
    const int64_t n = n0 + r < p.N ? n0 + r : p.N - 1;
    piece[CX + q] = ((lane & 7) ^ ((r & 3) | (r / (4 * NT) & 1) << 2)) * 16;
    src[CX + q] = p.w + n * p.K;
  }
  auto copy = [&](int64_t k0, int buf) {
#pragma unroll
    for (int q = 0; q < CX + CW; ++q) {
      const int64_t k = k0 + piece[q];
      const uint8_t* from = k < p.K ? src[q] + k : (const uint8_t*)&kZeros;
      const int row = q < CX ? (wave * CX + q) * 8 : BM + (wave * CW + q - CX) * 8;
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                       (__attribute__((address_space(3))) void*)&lds[buf][row * BK], 16, 0, 0);
    }
  };

  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int lr = lane & 15, lq = lane >> 4;
  auto fragment = [&](const uint8_t* base, int row, int key) {
    const uint8_t* r = base + row * BK;
    const i32x4 a = *(const i32x4*)(r + ((2 * lq) ^ key) * 16), b = *(const i32x4*)(r + ((2 * lq + 1) ^ key) * 16);
    return i32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  };
  copy(0, 0);
  int buf = 0;
  for (int64_t k0 = 0; k0 < p.K; k0 += BK, buf ^= 1) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // this wave's part of the slice has arrived
    __builtin_amdgcn_s_barrier();                      // everybody's has, and the other buffer is no longer read
    if (k0 + BK < p.K) copy(k0 + BK, buf ^ 1);
    const uint8_t *xs = lds[buf], *ws = lds[buf] + BM * BK;
    i32x8 wf[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      // lane row lr of tile j is row 4 NT (lr / 4) + 4 j + lr % 4 of the wave's: a lane's sums over all j are 4 NT consecutive n
      const int r = wn * NT * 16 + (lr >> 2) * 4 * NT + 4 * j + (lr & 3);
      wf[j] = fragment(ws, r, (r & 3) | (r / (4 * NT) & 1) << 2);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int r = (wm * MT + i) * 16 + lr;
      const i32x8 xf = fragment(xs, r, r & 7);
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] = mfma8(wf[j], xf, acc[i][j]);
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    float v[4 * NT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) v[4 * j + r] = acc[i][j][r];
    finish<T, 4 * NT>(p, m0 + (wm * MT + i) * 16 + lr, n0 + wn * NT * 16 + lq * 4 * NT, v);
  }
}

// ------------------------------------------------------------------------------------------------ few rows
// MT x 16 rows of x against 16 rows of w: the bytes of w bound it.  The waves of a workgroup take slices of 128 bytes of K in turn, straight
// from memory into the instruction's operands, and add their sums in LDS.
template <typename T, int MT, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void linear_rows_kernel(LinearParams p) {
  __shared__ f32x4 sums[WAVES][MT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15, lq = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int64_t n = n0 + lr < p.N ? n0 + lr : p.N - 1;
  const uint8_t* wr = p.w + n * p.K + lq * 32;
  const uint8_t* xr[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t m = i * 16 + lr < p.M ? i * 16 + lr : p.M - 1;
    xr[i] = p.x + m * p.K + lq * 32;
  }
  f32x4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int64_t slices = (p.K + 127) / 128, per = (slices + p.splits - 1) / p.splits;
  const int64_t first = blockIdx.y * per, end = first + per < slices ? first + per : slices;
  auto load = [&](const uint8_t* r, int64_t k) {
    // K in multiples of 16: a lane's 32 bytes end in the middle at most
    const i32x4 zero = {0, 0, 0, 0};
    const i32x4 a = k + lq * 32 < p.K ? *(const i32x4*)(r + k) : zero, b = k + lq * 32 + 16 < p.K ? *(const i32x4*)(r + k + 16) : zero;
    return i32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  };
  for (int64_t s = first + wave; s < end; s += WAVES) {
    const i32x8 wf = load(wr, s * 128);
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i] = mfma8(wf, load(xr[i], s * 128), acc[i]);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) sums[wave][i][lane] = acc[i];
  __syncthreads();
  for (int i = wave; i < MT; i += WAVES) {
    f32x4 t = sums[0][i][lane];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) t += sums[w][i][lane];
    const float v[4] = {t[0], t[1], t[2], t[3]};
    finish<T, 4>(p, i * 16 + lr, n0 + lq * 4, v);
  }
}

template <typename T, int BM, int BN, int WM, int WN>
int launch_tiles(const LinearParams& p, hipStream_t st) {
  const int64_t total = fla_cdiv(p.M, BM) * fla_cdiv(p.N, BN);
  FLA_REQUIRE(total <= 0x7fffffff, FLA_E_UNSUPPORTED);
  hipLaunchKernelGGL((linear_tile_kernel<T, BM, BN, WM, WN>), dim3((unsigned)total), dim3(WM * WN * 64), 0, st, p);
  FLA_CHECK_LAUNCH();
  return FLA_OK;
}
template <typename T, int MT>
int launch_rows(const LinearParams& p, hipStream_t st) {
  hipLaunchKernelGGL((linear_rows_kernel<T, MT, 8>), dim3((unsigned)fla_cdiv(p.N, 16), 1), dim3(512), 0, st, p);
  FLA_CHECK_LAUNCH();
  return FLA_OK;
}
template <typename T>
int launch_linear(const LinearParams& p, hipStream_t st) {
  if (p.M <= 16) return launch_rows<T, 1>(p, st);
  if (p.M <= 32) return launch_rows<T, 2>(p, st);
  if (p.M <= 48) return launch_rows<T, 3>(p, st);
  if (p.M <= 64) return launch_rows<T, 4>(p, st);
  const int64_t big = fla_cdiv(p.M, 256) * fla_cdiv(p.N, 256), mid = fla_cdiv(p.M, 128) * fla_cdiv(p.N, 128);
  if (big >= 192) return launch_tiles<T, 256, 256, 2, 4>(p, st);
  if (mid >= 128) return launch_tiles<T, 128, 128, 2, 2>(p, st);
  return launch_tiles<T, 64, 64, 2, 2>(p, st);
}

}  // namespace

extern "C" int fla_quant_linear(const void* x, const float* x_scale, const void* weight, const float* weight_scale, const void* bias,
                                int bias_dtype, const void* residual, int residual_dtype, void* y, int64_t M, int64_t N, int64_t K,
                                int activation, int dtype, fla_stream_t stream) {
  FLA_REQUIRE(x && x_scale && weight && weight_scale && y && M >= 0 && N > 0 && K > 0, FLA_E_INVALID);
  FLA_REQUIRE(activation >= FLA_ACT_NONE && activation <= FLA_ACT_RELU, FLA_E_INVALID);
  FLA_REQUIRE(dtype == FLA_BF16 || dtype == FLA_F16, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(!bias || bias_dtype == dtype || bias_dtype == FLA_F32, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(!residual || residual_dtype == dtype || residual_dtype == FLA_F32, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(K % 16 == 0 && N <= 0x7fffffff && M <= 0x7fffffff, FLA_E_UNSUPPORTED);
  FLA_REQUIRE((((uintptr_t)x) | ((uintptr_t)weight)) % 16 == 0, FLA_E_ALIGNMENT);
  if (M == 0) return FLA_OK;
  LinearParams p{};
  p.x = (const uint8_t*)x, p.sx = x_scale, p.w = (const uint8_t*)weight, p.sw = weight_scale, p.bias = bias, p.res = residual, p.y = y;
  p.M = M, p.N = N, p.K = K, p.act = activation, p.splits = 1;
  p.bias_f32 = bias_dtype == FLA_F32, p.res_f32 = residual_dtype == FLA_F32;
  p.wide = N % 8 == 0 && (((uintptr_t)residual) | ((uintptr_t)y)) % 16 == 0;
  hipStream_t st = (hipStream_t)stream;
  return dtype == FLA_BF16 ? launch_linear<bf16>(p, st) : launch_linear<f16>(p, st);
}
