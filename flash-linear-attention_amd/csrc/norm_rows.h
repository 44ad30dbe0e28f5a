// RMS norm and layer norm with the residual's addition in front of them, forward and backward, and an output in 8 bits with a scale per row:
//   s = x + r,   mu = mean s (RMS norm: 0),   rstd = 1 / sqrt(mean (s - mu)^2 + eps),   xh = (s - mu) rstd,   y = xh w (+ b)
//   8 bits:   scale = max(max|y|, 1e-30) / 448,   q = e4m3(y / scale);   as integers: / 127,   q = the whole number next to y / scale
//   ds = (w dy - mean(w dy) - xh mean(xh w dy)) rstd + ds_out (RMS norm: without mean(w dy)),   dw = sum dy xh,   db = sum dy
// HBM-streaming: every operand is read once and every result written once, a row stays in the registers of the lanes that hold
// it (8 elements a lane and pass), so that the squares are those of the centred elements: a mean far from zero costs no digits.  s is summed
// and normalised in fp32; what is kept of it (residual_out, in the residual's type) is what the backward reads, so xh there carries the
// rounding of the residual stream and no other.
#pragma once
#include <type_traits>

#include "fla_common.h"
#include "row_vec.h"

namespace {

constexpr float kE4M3Max = 448.f, kInt8Max = 127.f, kAmaxMin = 1e-30f;
enum Rows8 { kRowsNone = FLA_ROWS_NONE, kRowsE4M3 = FLA_ROWS_E4M3, kRowsInt8 = FLA_ROWS_INT8 };   // the output in 8 bits

struct NormParams {
  const void* x;        // [M,N]
  const void* res;      // [M,N] or NULL
  const void* w;        // [N] or NULL
  const void* b;        // [N] or NULL
  void* y;              // [M,N] (or the 8-bit rows)
  float* scale;         // [M], 8-bit rows only
  void* res_out;        // [M,N] or NULL
  float* rstd;          // [M] or NULL; backward: read
  float* mean;          // [M], layer norm: as rstd
  // backward: x is what the forward normalised
  const void* dy;
  const void* dres;     // [M,N] in the kept type, or NULL
  void* dx;
  void* dres_in;        // a copy of dx in the kept type, or NULL
  float* dw_part;       // [gridDim.x, N], rows part_ld apart, or NULL
  float* db_part;
  int64_t M, part_ld;
  int N;
  float eps;
  int res_f32, res_out_f32, w_f32, plain;   // plain: rows are not normalised (8-bit rows of x itself)
};

template <typename T, bool WIDE>
FLA_DEVICE void load8_of(const void* base, int f32, int64_t at, int valid, float* o) {
  if (f32) Row8<float>::unpack(load_raw8<float, WIDE>((const float*)base + at, valid), o);
  else Row8<T>::unpack(load_raw8<T, WIDE>((const T*)base + at, valid), o);
}
template <typename T, bool WIDE>
FLA_DEVICE void store8_of(void* base, int f32, int64_t at, int valid, const float* v) {
  if (f32) store8<float, WIDE>((float*)base + at, v, valid);
  else store8<T, WIDE>((T*)base + at, v, valid);
}

// Sum or maximum over the TPR threads that hold a row, in every one of them.  Rows of more than a wave go through LDS, `turn`
// alternating so that a value is not overwritten while another wave still reads it (one barrier an exchange).
enum RowJoin { kSum, kMax, kMaxOrNan };   // (kMax passes over NaN)
template <int JOIN>
FLA_DEVICE float row_join(float a, float b) {
  return JOIN == kSum ? a + b : JOIN == kMax ? fmaxf(a, b) : __builtin_elementwise_maximum(a, b);
}
template <int TPR, int JOIN>
FLA_DEVICE float row_reduce(float v, float (*lds)[TPR > 64 ? TPR / 64 : 1], int turn) {
  constexpr int W = TPR < 64 ? TPR : 64;
#pragma unroll
  for (int m = W / 2; m >= 1; m >>= 1) v = row_join<JOIN>(v, __shfl_xor(v, m, 64));
  if (TPR > 64) {
    if ((threadIdx.x & 63) == 0) lds[turn][threadIdx.x % TPR >> 6] = v;
    lds_barrier();
    v = lds[turn][0];
#pragma unroll
    for (int i = 1; i < (TPR > 64 ? TPR / 64 : 1); ++i) v = row_join<JOIN>(v, lds[turn][i]);
  }
  return v;
}
// two sums with one exchange
template <int TPR>
FLA_DEVICE f32x2 row_sum2(f32x2 v, f32x2 (*lds)[TPR > 64 ? TPR / 64 : 1], int turn) {
  constexpr int W = TPR < 64 ? TPR : 64;
#pragma unroll
  for (int m = W / 2; m >= 1; m >>= 1) v += f32x2{__shfl_xor(v[0], m, 64), __shfl_xor(v[1], m, 64)};
  if (TPR > 64) {
    if ((threadIdx.x & 63) == 0) lds[turn][threadIdx.x % TPR >> 6] = v;
    lds_barrier();
    v = lds[turn][0];
#pragma unroll
    for (int i = 1; i < (TPR > 64 ? TPR / 64 : 1); ++i) v += lds[turn][i];
  }
  return v;
}

// Eight elements in 8 bits, of which the first `valid` exist.  They are divided, as the scale is defined: a product with its rounded reciprocal
// moves values next to a border of the 8-bit type.
template <int ROWS8, bool WIDE>
FLA_DEVICE void store_rows8(uint8_t* at, const float* v, float scale, int valid) {
  int pk[2] = {0, 0};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (ROWS8 == kRowsE4M3) {
      pk[h] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h] / scale, v[4 * h + 1] / scale, pk[h], false);
      pk[h] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h + 2] / scale, v[4 * h + 3] / scale, pk[h], true);
    } else {   // (the quotient is at most 127 and a few units of fp32; of NaN and infinite rows the scale says so, the whole numbers are 0)
#pragma unroll
      for (int i = 0; i < 4; ++i) pk[h] |= ((int)__builtin_rintf(v[4 * h + i] / scale) & 0xff) << (8 * i);
    }
  }
  if (WIDE) {
    if (valid > 0) *(int2*)at = int2{pk[0], pk[1]};
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (i < valid) at[i] = (uint8_t)(pk[i / 4] >> (8 * (i % 4)));
  }
}
// the maximum as it is joined, and the scale of a row from it; a row of integers that holds NaN has the scale NaN (e4m3 keeps the element's own)
template <int ROWS8>
constexpr int kAmaxJoin = ROWS8 == kRowsInt8 ? kMaxOrNan : kMax;
template <int ROWS8>
FLA_DEVICE float rows8_scale(float amax) { return row_join<kAmaxJoin<ROWS8>>(amax, kAmaxMin) / (ROWS8 == kRowsInt8 ? kInt8Max : kE4M3Max); }

// A row for TPR threads, NP passes of 8 elements each; MEAN: the layer norm.
template <typename T, int TPR, int NP, bool WIDE, bool MEAN, int ROWS8>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void norm_fwd_kernel(NormParams p) {
  constexpr int BLOCK = TPR > 256 ? TPR : 256, RPB = BLOCK / TPR;
  __shared__ float lds[3][TPR > 64 ? TPR / 64 : 1];
  const int sub = threadIdx.x % TPR, N = p.N;
  const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
  if (row >= p.M) return;      // (all threads of a row together; a row of several waves is a block's only one)
  float v[NP][VEC];
  float ss = 0.f;
#pragma unroll
  for (int q = 0; q < NP; ++q) {
    const int col = (q * TPR + sub) * VEC, valid = N - col;
    load8_of<T, WIDE>(p.x, 0, row * N + col, valid, v[q]);
  }
  if (p.res) {
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      const int col = (q * TPR + sub) * VEC, valid = N - col;
      float r[VEC];
      load8_of<T, WIDE>(p.res, p.res_f32, row * N + col, valid, r);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[q][i] += r[i];
    }
  }
#pragma unroll
  for (int q = 0; q < NP; ++q) {
    const int col = (q * TPR + sub) * VEC, valid = N - col;
    if (p.res_out) store8_of<T, WIDE>(p.res_out, p.res_out_f32, row * N + col, valid, v[q]);
#pragma unroll
    for (int i = 0; i < VEC; ++i) ss = MEAN ? ss + v[q][i] : fmaf(v[q][i], v[q][i], ss);
  }
  if (MEAN) {
    const float mean = row_reduce<TPR, kSum>(ss, lds, 2) / (float)N;
    if (p.mean && sub == 0) p.mean[row] = mean;
    ss = 0.f;
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      const int valid = N - (q * TPR + sub) * VEC;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        v[q][i] = (WIDE ? valid > 0 : i < valid) ? v[q][i] - mean : 0.f;
        ss = fmaf(v[q][i], v[q][i], ss);
      }
    }
  }
  float rstd = 1.f;
  if (MEAN || !p.plain) {
    rstd = rsqrtf(row_reduce<TPR, kSum>(ss, lds, 0) / (float)N + p.eps);
    if (p.rstd && sub == 0) p.rstd[row] = rstd;
  }
  float amax = 0.f;
#pragma unroll
  for (int q = 0; q < NP; ++q) {
    const int col = (q * TPR + sub) * VEC, valid = N - col;
    float w[VEC], b[VEC];
    if (p.w) load8_of<T, WIDE>(p.w, p.w_f32, col, valid, w);
    if (p.b) load8_of<T, WIDE>(p.b, p.w_f32, col, valid, b);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      v[q][i] *= rstd;
      if (p.w) v[q][i] *= w[i];
      if (p.b) v[q][i] += b[i];
      if (ROWS8) amax = row_join<kAmaxJoin<ROWS8>>(amax, __builtin_fabsf(v[q][i]));
    }
    if (!ROWS8) store8<T, WIDE>((T*)p.y + row * N + col, v[q], valid);
  }
  if (ROWS8) {
    const float scale = rows8_scale<ROWS8>(row_reduce<TPR, kAmaxJoin<ROWS8>>(amax, lds, 1));
    if (sub == 0) p.scale[row] = scale;
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      const int col = (q * TPR + sub) * VEC;
      store_rows8<ROWS8, WIDE>((uint8_t*)p.y + row * N + col, v[q], scale, N - col);
    }
  }
}

// Rows in 8 bits of more elements than registers hold: the row's maximum, then its quotients from a second reading (out of L2: a workgroup's row
// is its own).  Rows of 28672 in bf16 (us): 32 in 6.4, 512 in 13, 8192 in 188, 3.75 TB/s (8192 of 16384, in registers: 90, 4.45).
constexpr int kLongThreads = 1024;
template <typename T, bool WIDE, int ROWS8>
__global__ __launch_bounds__(kLongThreads) void rows8_long_kernel(NormParams p) {
  __shared__ float lds[2][kLongThreads / 64];
  const int N = p.N;
  const int64_t row = blockIdx.x;
  const T* x = (const T*)p.x + row * N;
  float amax = 0.f;
#pragma unroll 4
  for (int col = threadIdx.x * VEC; col < N; col += kLongThreads * VEC) {
    float v[VEC];
    Row8<T>::unpack(load_raw8<T, WIDE>(x + col, N - col), v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) amax = row_join<kAmaxJoin<ROWS8>>(amax, __builtin_fabsf(v[i]));
  }
  const float scale = rows8_scale<ROWS8>(row_reduce<kLongThreads, kAmaxJoin<ROWS8>>(amax, lds, 0));
  if (threadIdx.x == 0) p.scale[row] = scale;
#pragma unroll 4
  for (int col = threadIdx.x * VEC; col < N; col += kLongThreads * VEC) {
    float v[VEC];
    Row8<T>::unpack(load_raw8<T, WIDE>(x + col, N - col), v);
    store_rows8<ROWS8, WIDE>((uint8_t*)p.y + row * N + col, v, scale, N - col);
  }
}

// Threads of a backward's workgroup: as many rows as 1024 threads hold where a row has waves of its own, so that their column sums meet in LDS and
// few partial sums are left for the launch that adds them (16384 x 2048: 4 us instead of 8.4 from workgroups of one row).
constexpr int bwd_block(int tpr) { return tpr <= 64 ? 256 : 1024; }

// Rows are walked so that the column sums of the weight gradients stay in registers and leave once per workgroup.  The operands of the next
// row are on their way while one is worked on.
template <typename T, typename KT, int TPR, int NP, bool WIDE, bool BIAS, bool MEAN>
__global__ __launch_bounds__(bwd_block(TPR)) void norm_bwd_kernel(NormParams p) {
  constexpr int BLOCK = bwd_block(TPR), RPB = BLOCK / TPR;
  __shared__ typename std::conditional<MEAN, f32x2, float>::type lds[RPB][2][TPR > 64 ? TPR / 64 : 1];
  __shared__ float sum[RPB > 1 ? RPB : 1][RPB > 1 ? TPR * VEC : 1];
  const int sub = threadIdx.x % TPR, rl = threadIdx.x / TPR, N = p.N;
  float dw[NP][VEC], db[NP][VEC];
#pragma unroll
  for (int q = 0; q < NP; ++q)
#pragma unroll
    for (int i = 0; i < VEC; ++i) dw[q][i] = db[q][i] = 0.f;
  int turn = 0;
  const float inv = 1.f / (float)N;
  const int64_t step = (int64_t)gridDim.x * RPB;
  typename Row8<KT>::raw ns[NP], nr[NP];
  typename Row8<T>::raw nd[NP];
  float nrstd, nmean = 0.f;
  auto fetch = [&](int64_t row) {
    const bool in = row < p.M;
    nrstd = in ? p.rstd[row] : 0.f;
    if (MEAN) nmean = in ? p.mean[row] : 0.f;
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      const int col = (q * TPR + sub) * VEC, valid = in ? N - col : 0;
      ns[q] = load_raw8<KT, WIDE>((const KT*)p.x + row * N + col, valid);
      nd[q] = load_raw8<T, WIDE>((const T*)p.dy + row * N + col, valid);
      if (p.dres) nr[q] = load_raw8<KT, WIDE>((const KT*)p.dres + row * N + col, valid);
    }
  };
  constexpr bool AHEAD = NP == 1;   // (the registers of two passes do not hold a second row)
  if (AHEAD) fetch((int64_t)blockIdx.x * RPB + rl);
  // every thread makes as many rounds: rows of several waves exchange through a barrier
  for (int64_t row0 = (int64_t)blockIdx.x * RPB; row0 < p.M; row0 += step, turn ^= 1) {
    const int64_t row = row0 + rl;
    if (!AHEAD) fetch(row);
    float s[NP][VEC], d[NP][VEC];
    typename Row8<KT>::raw r8[NP];
    const float rstd = nrstd, mean = nmean;
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      Row8<KT>::unpack(ns[q], s[q]);
      Row8<T>::unpack(nd[q], d[q]);
      r8[q] = nr[q];
    }
    if (AHEAD) fetch(row + step);
    float c = 0.f, c1 = 0.f;
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      const int col = (q * TPR + sub) * VEC;
      float w[VEC];
      if (p.w) load8_of<T, WIDE>(p.w, p.w_f32, col, N - col, w);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        // (behind the end of a row d and w are 0, and so are their sums)
        s[q][i] = MEAN ? (s[q][i] - mean) * rstd : s[q][i] * rstd;
        dw[q][i] = fmaf(d[q][i], s[q][i], dw[q][i]);
        if (BIAS) db[q][i] += d[q][i];
        if (p.w) d[q][i] *= w[i];
        c = fmaf(d[q][i], s[q][i], c);
        if (MEAN) c1 += d[q][i];
      }
    }
    if constexpr (MEAN) {
      const f32x2 both = row_sum2<TPR>(f32x2{c, c1}, lds[rl], turn);
      c = both[0] * inv, c1 = both[1] * inv;
    } else {
      c = row_reduce<TPR, kSum>(c, lds[rl], turn) * inv;
    }
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      const int col = (q * TPR + sub) * VEC, valid = row < p.M ? N - col : 0;
      float r[VEC];
      if (p.dres) Row8<KT>::unpack(r8[q], r);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        d[q][i] = (MEAN ? d[q][i] - c1 - s[q][i] * c : d[q][i] - s[q][i] * c) * rstd;
        if (p.dres) d[q][i] += r[i];
      }
      store8<T, WIDE>((T*)p.dx + row * N + col, d[q], valid);
      if (p.dres_in) store8<KT, WIDE>((KT*)p.dres_in + row * N + col, d[q], valid);
    }
  }
  for (int which = 0; which < (BIAS ? 2 : 1); ++which) {
    float* part = which ? p.db_part : p.dw_part;
    if (!part) continue;   // uniform
    part += (int64_t)blockIdx.x * p.part_ld;
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      const float* mine = which ? db[q] : dw[q];
      const int col = (q * TPR + sub) * VEC;
      if (RPB == 1) {
        store8<float, WIDE>(part + col, mine, N - col);
      } else {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum[rl][sub * VEC + i] = mine[i];
        __syncthreads();
        for (int k = threadIdx.x; k < TPR * VEC; k += BLOCK) {
          float t = 0.f;
#pragma unroll
          for (int r = 0; r < RPB; ++r) t += sum[r][k];
          if (q * TPR * VEC + k < N) part[q * TPR * VEC + k] = t;
        }
      }
    }
  }
}

// (threads to a row, passes) by the row's length.  Forward: a wave to a row up to 2048 elements (16384 rows in 54 us, 4.95 TB/s), but four
// waves where there are few rows (32 rows of 2048 to 8 bits: 4.0 us, with one wave 5.5).  Backward: rows of one pass as long as there are
// threads, since the column sums and the next row's operands take registers (16384 rows of 2048: 54 us; with four passes of a wave 75 us,
// 80 with the next row's operands in flight), and the least threads that hold them: 2^25 elements with the weight's gradient take 51 - 55 us (the bytes: 52)
// in rows of 64 to 16384, up to 63 where a quarter of the threads is idle (1024 in 256 threads: 67; 8192 in two passes of 512: 74, 16384 in four: 112).  The workgroups
// of 1024 threads have 128 registers: above 8192 elements with a bias 12 - 74 of them are spilled, with an fp32 stream alone 2 - 8, and with a bias and
// an fp32 stream 2 - 5 in rows of one pass from 1025 elements on; the others spill none.
#define NORM_FWD_SHAPES(CALL)                       \
  if (N <= 64) CALL(8, 1)                          \
  else if (N <= 128) CALL(16, 1)                   \
  else if (N <= 256) CALL(32, 1)                   \
  else if (N <= 512) CALL(64, 1)                   \
  else if (N <= 2048 && all.M <= kFewRows) CALL(256, 1) \
  else if (N <= 1024) CALL(64, 2)                  \
  else if (N <= 2048) CALL(64, 4)                  \
  else if (N <= 4096) CALL(256, 2)                 \
  else if (N <= 8192) CALL(256, 4)                 \
  else CALL(512, 4)
#define NORM_BWD_SHAPES(CALL)       \
  if (N <= 64) CALL(8, 1)          \
  else if (N <= 128) CALL(16, 1)   \
  else if (N <= 256) CALL(32, 1)   \
  else if (N <= 512) CALL(64, 1)   \
  else if (N <= 1024) CALL(128, 1) \
  else if (N <= 2048) CALL(256, 1) \
  else if (N <= 4096) CALL(512, 1) \
  else if (N <= 8192) CALL(1024, 1) \
  else CALL(1024, 2)

// Layer norm, bf16 with residual and bias: 16384 rows of 2048 forward 54 - 56 us (4.9 TB/s), backward 59 - 61 (4.5), 4.9 for the launch that adds the partial sums of both gradients.
// Its backward spills registers in unaligned rows: 2 - 17 in one pass with an fp32 stream, 1 - 70 in two passes (above 8192 elements).
constexpr int64_t kFewRows = 1024;
constexpr int64_t kMaxN = 512 * 4 * VEC;         // of rows that stay in registers
constexpr int64_t kMaxRow8 = 1 << 23;            // of rows that are brought to 8 bits and nothing else: as many as the product takes
int bwd_rows_per_block(int64_t N) {
  return N <= 64 ? 32 : N <= 128 ? 16 : N <= 256 ? 8 : N <= 512 ? 4 : N <= 1024 ? 8 : N <= 2048 ? 4 : N <= 4096 ? 2 : 1;
}
// as many workgroups as are on the chip at once: 16 waves a CU
int64_t bwd_workgroups(int64_t N) { return N <= 512 ? 1024 : 256; }

constexpr int64_t kLaunchRows = 1 << 22;   // of a forward launch: one is less than 2^32 threads

// the `rows` rows from number `row` on
template <typename T, int ROWS8>
NormParams rows_from(const NormParams& all, int64_t row, int64_t rows) {
  NormParams p = all;
  const int64_t at = row * p.N;
  p.x = (const T*)p.x + at;
  if (p.res) p.res = (const char*)p.res + at * (p.res_f32 ? 4 : sizeof(T));
  if (p.res_out) p.res_out = (char*)p.res_out + at * (p.res_out_f32 ? 4 : sizeof(T));
  p.y = (char*)p.y + at * (ROWS8 ? 1 : sizeof(T));
  if (p.scale) p.scale += row;
  if (p.mean) p.mean += row;
  if (p.rstd) p.rstd += row;
  p.M = rows;
  return p;
}
template <typename T, bool WIDE, bool MEAN, int ROWS8>
int launch_fwd(const NormParams& all, hipStream_t st) {
  const int N = all.N;
  if constexpr (ROWS8 != kRowsNone && !MEAN) {
    if (N > kMaxN) {
      constexpr int64_t most = kLaunchRows / 2;
      for (int64_t row = 0; row < all.M; row += most) {
        const NormParams p = rows_from<T, ROWS8>(all, row, all.M - row < most ? all.M - row : most);
        hipLaunchKernelGGL((rows8_long_kernel<T, WIDE, ROWS8>), dim3((unsigned)p.M), dim3(kLongThreads), 0, st, p);
        FLA_CHECK_LAUNCH();
      }
      return FLA_OK;
    }
  }
  for (int64_t row = 0; row < all.M; row += kLaunchRows) {
    const NormParams p = rows_from<T, ROWS8>(all, row, all.M - row < kLaunchRows ? all.M - row : kLaunchRows);
#define CALL(TPR, NP)                                                                                                             \
  {                                                                                                                               \
    constexpr int block = TPR > 256 ? TPR : 256;                                                                                  \
    hipLaunchKernelGGL((norm_fwd_kernel<T, TPR, NP, WIDE, MEAN, ROWS8>), dim3((unsigned)fla_cdiv(p.M, block / TPR)), dim3(block), 0, st, p); \
  }
    NORM_FWD_SHAPES(CALL)
#undef CALL
    FLA_CHECK_LAUNCH();
  }
  return FLA_OK;
}
template <typename T, typename KT, bool WIDE, bool MEAN>
int launch_bwd(const NormParams& p, int grid, hipStream_t st) {
  const int N = p.N;
#define CALL(TPR, NP)                                                                                                                       \
  {                                                                                                                                         \
    constexpr int block = bwd_block(TPR);                                                                                               \
    if (p.db_part) hipLaunchKernelGGL((norm_bwd_kernel<T, KT, TPR, NP, WIDE, true, MEAN>), dim3(grid), dim3(block), 0, st, p);                     \
    else hipLaunchKernelGGL((norm_bwd_kernel<T, KT, TPR, NP, WIDE, false, MEAN>), dim3(grid), dim3(block), 0, st, p);                              \
  }
  NORM_BWD_SHAPES(CALL)
#undef CALL
  FLA_CHECK_LAUNCH();
  return FLA_OK;
}
// whether rows of N elements behind each of the pointers can be read 16 bytes at a time
bool wide(int64_t N, std::initializer_list<const void*> ps) {
  uintptr_t any = 0;
  for (const void* p : ps) any |= (uintptr_t)p;
  return any % 16 == 0 && N % VEC == 0;
}
bool type_ok(int t, int dtype) { return t == dtype || t == FLA_F32; }

template <bool MEAN>
int norm_forward(const void* x, const void* residual, int residual_dtype, const void* weight, const void* bias, int weight_dtype, void* y,
                 float* scale, void* residual_out, int residual_out_dtype, float* mean, float* rstd, int64_t M, int64_t N, float eps,
                 int normalise, int rows8, int dtype, fla_stream_t stream) {
  FLA_REQUIRE(x && y && M >= 0 && N > 0 && (normalise || (!weight && !bias && !rstd)), FLA_E_INVALID);
  FLA_REQUIRE(rows8 >= FLA_ROWS_NONE && rows8 <= FLA_ROWS_INT8 && (rows8 != FLA_ROWS_NONE) == (scale != nullptr), FLA_E_INVALID);
  FLA_REQUIRE(normalise || scale, FLA_E_INVALID);
  const bool rows_only = !normalise && !residual && !residual_out;
  FLA_REQUIRE(N <= (rows_only ? kMaxRow8 : kMaxN) && M <= 0x7fffffffLL, FLA_E_UNSUPPORTED);
  FLA_REQUIRE(!residual || type_ok(residual_dtype, dtype), FLA_E_UNSUPPORTED);
  FLA_REQUIRE(!residual_out || type_ok(residual_out_dtype, dtype), FLA_E_UNSUPPORTED);
  FLA_REQUIRE((!weight && !bias) || type_ok(weight_dtype, dtype), FLA_E_UNSUPPORTED);
  if (M == 0) return FLA_OK;
  NormParams p{};
  p.x = x, p.res = residual, p.w = weight, p.b = bias, p.y = y, p.scale = scale, p.res_out = residual_out, p.rstd = rstd, p.mean = mean;
  p.M = M, p.N = (int)N, p.eps = eps, p.plain = !normalise;
  p.res_f32 = residual_dtype == FLA_F32, p.res_out_f32 = residual_out_dtype == FLA_F32, p.w_f32 = weight_dtype == FLA_F32;
  const bool w = wide(N, {x, residual, weight, bias, y, residual_out});
  hipStream_t st = (hipStream_t)stream;
#define R_(T, ROWS8) return w ? launch_fwd<T, true, MEAN, ROWS8>(p, st) : launch_fwd<T, false, MEAN, ROWS8>(p, st);
#define D_(E, T)                               \
  if (dtype == E) {                            \
    if (rows8 == kRowsE4M3) R_(T, kRowsE4M3)   \
    if (rows8 == kRowsInt8) R_(T, kRowsInt8)   \
    R_(T, kRowsNone)                           \
  }
  D_(FLA_BF16, bf16)
  D_(FLA_F16, f16)
  D_(FLA_F32, float)
#undef D_
#undef R_
  return FLA_E_UNSUPPORTED;
}

int norm_workgroups(int64_t M, int64_t N) {
  if (M <= 0 || N <= 0) return 1;
  const int64_t g = fla_cdiv(M, bwd_rows_per_block(N));
  const int64_t most = bwd_workgroups(N);
  return (int)(g < most ? g : most);
}

template <bool MEAN>
int norm_backward(const void* dy, const void* kept, int kept_dtype, const void* weight, int weight_dtype, const float* mean, const float* rstd,
                  const void* dresidual, void* dx, void* dresidual_in, float* dw_partial, float* db_partial, int64_t partial_ld, int64_t M, int64_t N,
                  int dtype, fla_stream_t stream) {
  FLA_REQUIRE(dy && kept && rstd && dx && (!MEAN || mean) && M >= 0 && N > 0, FLA_E_INVALID);
  FLA_REQUIRE(N <= kMaxN && M <= 0x7fffffffLL && type_ok(kept_dtype, dtype), FLA_E_UNSUPPORTED);
  FLA_REQUIRE(!weight || type_ok(weight_dtype, dtype), FLA_E_UNSUPPORTED);
  FLA_REQUIRE(partial_ld >= N, FLA_E_INVALID);
  const bool w = wide(N, {dy, kept, weight, dresidual, dx, dresidual_in});
  FLA_REQUIRE(((uintptr_t)dw_partial | (uintptr_t)db_partial | (w ? (uintptr_t)(partial_ld * 4) : 0)) % (w ? 16 : 4) == 0, FLA_E_ALIGNMENT);
  if (M == 0) return FLA_OK;
  NormParams p{};
  p.x = kept, p.w = weight, p.rstd = (float*)rstd, p.mean = (float*)mean, p.dy = dy, p.dres = dresidual, p.dx = dx, p.dres_in = dresidual_in;
  p.dw_part = dw_partial, p.db_part = db_partial, p.part_ld = partial_ld, p.M = M, p.N = (int)N;
  p.w_f32 = weight_dtype == FLA_F32;
  const int grid = norm_workgroups(M, N);
  hipStream_t st = (hipStream_t)stream;
#define D_(E, T)                                                                                                                            \
  if (dtype == E && kept_dtype == E) return w ? launch_bwd<T, T, true, MEAN>(p, grid, st) : launch_bwd<T, T, false, MEAN>(p, grid, st);     \
  if (dtype == E) return w ? launch_bwd<T, float, true, MEAN>(p, grid, st) : launch_bwd<T, float, false, MEAN>(p, grid, st);
  D_(FLA_BF16, bf16)
  D_(FLA_F16, f16)
  D_(FLA_F32, float)
#undef D_
  return FLA_E_UNSUPPORTED;
}

}  // namespace
