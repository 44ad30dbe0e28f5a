// Products with few rows of x:  c[m,n] = sum_k x[m,k] w[n,k]  for at most MT x 16 rows m and 16 rows n of one matrix w, or of each of two.
// The bytes of w bound it, and those of x out of L2 from 32 rows on.  The waves take slices of 128 bytes of k in turn, each through RING pieces of LDS of
// its own, waiting for nobody until the sums are added in the waves' order.
// Measured (bf16, two weights, out of HBM, in a captured graph): 1 x 4096 to 11008 37.4 us (4.8 TB/s of the weights), 16 rows 38.3, 32 42.9, 48 45.8, 64 51.9 (x comes once for
// every 16 columns: at 64 rows twice the weights' bytes); 1 x 2048 to 5632 12.1.  One or two waves a workgroup and rings of three and four were none faster.
#pragma once
#include "matrix_tiles.h"

namespace {

template <typename T>
struct Mat16 {   // 16 bytes of 16 rows each
  typedef f32x4 acc;
  static FLA_DEVICE acc mma(i32x4 a, i32x4 b, acc c) {
    typedef typename Elem<T>::v8 v8;
    return Elem<T>::mfma16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c);
  }
};
template <>
struct Mat16<int8_t> {
  typedef i32x4 acc;
  static FLA_DEVICE acc mma(i32x4 a, i32x4 b, acc c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }
};

template <typename T, int MT, int MATS, int WAVES, int RING>
struct MatPanel {
  typedef typename Mat16<T>::acc acc_t;
  static constexpr int kRows = (MT + MATS) * 16, kPiece = kRows * kSliceBytes, kCopies = kRows / 8;   // rows of x, then those of each w
  static constexpr int kLds = WAVES * RING * kPiece > WAVES * MATS * MT * 1024 ? WAVES * RING * kPiece : WAVES * MATS * MT * 1024;

  // f(matrix-wise sums, i): row tile i of this wave's; lane l holds sums[w][r] of m = 16 i + l % 16 and n = 4 (l / 16) + r.  x of M rows, w[] from row n0 on
  // with N rows left; pitch: bytes of a row, a multiple of 16.
  template <typename F>
  static FLA_DEVICE void run(char* lds, const char* x, int64_t M, const char* const (&w)[MATS], int64_t N, int pitch, const F& f) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 15, lq = lane >> 4;
    const int piece = ((lane & 7) ^ (lane >> 3)) * 16;
    __amdgpu_buffer_rsrc_t from[1 + MATS];
    from[0] = MatSource{x, x + M * pitch, 0}.descriptor();
#pragma unroll
    for (int i = 0; i < MATS; ++i) from[1 + i] = MatSource{w[i], w[i] + (N < 16 ? N : 16) * pitch, 0}.descriptor();
    const uint32_t at = (uint32_t)(lane >> 3) * pitch + piece;
    char* mine = lds + wave * RING * kPiece;
    auto copy = [&](int k0, int buf) {   // slices beyond the end are zeros
      const uint32_t here = piece + k0 < pitch ? at + k0 : kMatBeyond;
#pragma unroll
      for (int q = 0; q < kCopies; ++q) {
        const int r = q < 2 * MT ? q : (q - 2 * MT) % 2;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(from[q < 2 * MT ? 0 : 1 + (q - 2 * MT) / 2],
                                                 (__attribute__((address_space(3))) void*)(mine + buf * kPiece + q * 8 * kSliceBytes), 16,
                                                 here == kMatBeyond ? (int)kMatBeyond : (int)(here + r * 8 * pitch), 0, 0, 0);
      }
    };
    auto fragment = [&](int buf, int row, int h) {   // 16-byte pieces keyed by the row: sixteen lanes meet all banks once
      return *(const i32x4*)(mine + buf * kPiece + row * kSliceBytes + (((4 * h + lq) ^ (row & 7)) * 16));
    };
    acc_t acc[MATS][MT];
#pragma unroll
    for (int i = 0; i < MATS; ++i)
#pragma unroll
      for (int j = 0; j < MT; ++j) acc[i][j] = acc_t{};
#pragma unroll
    for (int d = 0; d + 1 < RING; ++d) copy((wave + d * WAVES) * kSliceBytes, d);
    int buf = 0;
    for (int k0 = wave * kSliceBytes; k0 < pitch; k0 += WAVES * kSliceBytes) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the slice that the next copy replaces has been read
      copy(k0 + (RING - 1) * WAVES * kSliceBytes, buf ? buf - 1 : RING - 1);
      asm volatile("s_waitcnt vmcnt(%0)" ::"i"((RING - 1) * kCopies) : "memory");   // (loads arrive in order: this slice has)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        i32x4 wf[MATS];
#pragma unroll
        for (int i = 0; i < MATS; ++i) wf[i] = fragment(buf, (MT + i) * 16 + lr, h);
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          const i32x4 xf = fragment(buf, j * 16 + lr, h);
#pragma unroll
          for (int i = 0; i < MATS; ++i) acc[i][j] = Mat16<T>::mma(wf[i], xf, acc[i][j]);
        }
      }
      buf = buf + 1 < RING ? buf + 1 : 0;
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __syncthreads();
    acc_t(*sums)[MATS][MT][64] = (acc_t(*)[MATS][MT][64])lds;
#pragma unroll
    for (int i = 0; i < MATS; ++i)
#pragma unroll
      for (int j = 0; j < MT; ++j) sums[wave][i][j][lane] = acc[i][j];
    __syncthreads();
    for (int j = wave; j < MT; j += WAVES) {
      acc_t t[MATS];
#pragma unroll
      for (int i = 0; i < MATS; ++i) {
        t[i] = sums[0][i][j][lane];
#pragma unroll
        for (int v = 1; v < WAVES; ++v) t[i] += sums[v][i][j][lane];
      }
      f(t, j);
    }
  }
};

}  // namespace
