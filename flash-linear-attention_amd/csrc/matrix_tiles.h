// Tiles of a matrix product  c[m,n] = sum_k a(m,k) b(n,k)  on the 32x32 matrix instructions, each operand with its contraction index
// contiguous (rows [m][k]) or strided (rows [k][m]), 16-bit elements or 8-bit integers, sums in 32 bits.
//
// Four waves share a BM x BN tile, a wave holds a quarter of it (MT x NT tiles of 32 x 32) and, where the tile is 256 x 256, has a SIMD's
// registers to itself.  Slices of 128 bytes of k travel straight from memory into a ring of RING pieces of LDS.  While one half of a slice is
// multiplied, the fragments of the next half are read; one barrier a slice, ahead of its second half, orders everything: behind it the next slice is
// there for every wave, and as everybody's fragments of this one are in registers its piece is free.
//
// A wave's quarter of 128 x 128 reads 32 fragments for 64 instructions: 128 KB a slice and CU, half of what LDS passes in that time.  (Eight waves
// of 128 x 64 read 192 KB, which with the 64 KB of the copies is all of it.)
//
// Measured (bf16): 8192^3 812 us, 1.35 PFLOP/s (torch 706 - 717; with the contraction strided in both operands 810 - 817, torch 949 - 960), 8192 x 11264 x 2048 340 us (torch 395),
// 8192 x 2048 x 11264 with it strided in one 296 (torch 329), 5632 x 2048 x 8192 with it strided in both 178 (torch 207 - 214).  The card holds 1.55 GHz under 8192^3
// (GRBM_GUI_ACTIVE); of 1.37M cycles 1.05M are matrix instructions.  With copies of the same lines again and again it takes 1.21M: what is lost is memory's side.
// Tried and slower or no faster: the 16x16 instruction (the compiler moves accumulators between the loops' registers), slices of 64 bytes in rings of three to five (of 1.41M cycles
// copies and LDS reads cost 0.22M), pointers instead of descriptors (three vector instructions a copy), a barrier every second slice, copies that the waves issue in turn,
// a load a line some slices ahead (L2), a ring of three for one operand.
//
// Memory is read through buffer descriptors that end where the operand ends: rows and pieces behind it are zeros, by the hardware's range check.
#pragma once
#include "fla_common.h"

namespace {

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// 16 bytes of a row of the operands and the instruction that takes them
template <typename T>
struct Mat {   // bf16, f16
  typedef f32x16 acc;
  static FLA_DEVICE acc mma(i32x4 a, i32x4 b, acc c) {
    typedef typename Elem<T>::v8 v8;
    return Elem<T>::mfma32(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c);
  }
};
template <>
struct Mat<int8_t> {
  typedef i32x16 acc;
  static FLA_DEVICE acc mma(i32x4 a, i32x4 b, acc c) { return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0); }
};

// The transposing read of four rows.  __restrict__ gives the access an alias scope: of one without any the compiler takes it that it may read what copies
// in flight write, and waits for all of them ahead of every read.  (The tiles wait where it is needed.)
FLA_DEVICE s16x4 lds_read_tr(lds_s16x4* __restrict__ p) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16(p); }

constexpr int kSliceBytes = 128;          // of k
constexpr uint32_t kMatBeyond = 1u << 31; // an offset that no descriptor reaches
constexpr int64_t kMatMaxDim = 1 << 22;   // elements of a row of an operand: 256 rows are less than 2^31 bytes

// From where on a slice is read, and to where the operand goes
struct MatSource {
  const char *from, *end;
  int left;   // of k, in bytes (contiguous operands)
  FLA_DEVICE __amdgpu_buffer_rsrc_t descriptor() const {
    const int64_t bytes = end - from;
    return __builtin_amdgcn_make_buffer_rsrc((void*)from, 0, bytes < 0 ? 0 : bytes < (int64_t)kMatBeyond - 1 ? (int)bytes : (int)(kMatBeyond - 1), 0x00027000);
  }
};
FLA_DEVICE void mat_copy(__amdgpu_buffer_rsrc_t from, uint32_t at, char* lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void*)lds, 16, (int)at, 0, 0, 0);
}

// One operand of a tile, ROWS of it; STRIDED: rows of memory are [k][ROWS], otherwise [ROWS][k].  PAIR: rows of two matrices, 32 of the one and 32 of the
// other in turn (the products of one row with both are then in one lane).
//
// LDS layout of a slice.  Contiguous: ROWS rows of 128 bytes, the 16-byte pieces of a row permuted by a key of the row.  A b128 read serves lanes
// 0-3, 12-15, 20-27 together, then 4-11, 16-19, 28-31, and the same of the upper half: with these keys each sixteen meet all 64 banks once.
// Strided (16-bit types): 64 rows of ROWS elements, their 64-byte quarters permuted by a key of k.  The transposing read takes 64 bytes of each of four
// rows for 32 lanes, which the keys spread over all banks.
template <int ROWS, bool STRIDED, bool PAIR = false>
struct Operand;

template <int ROWS, bool PAIR>
struct Operand<ROWS, false, PAIR> {
  static constexpr int kSources = PAIR ? 2 : 1, kBytes = ROWS * kSliceBytes, kCopies = ROWS / 32;   // copy instructions of each of four waves for a slice
  static_assert(kCopies >= 1, "whole copies");
  static FLA_DEVICE int key(int r) { return (r >> 1 & 1) | (r >> 3 & 3) << 1; }
  uint32_t at[kCopies];
  int piece[kCopies];      // bytes of k ahead of what this lane copies
  FLA_DEVICE void start(int wave, int lane, uint32_t pitch) {
#pragma unroll
    for (int q = 0; q < kCopies; ++q) {
      const int r = (wave * kCopies + q) * 8 + (lane >> 3);
      piece[q] = ((lane & 7) ^ key(r)) * 16;
      at[q] = (uint32_t)(PAIR ? r / 64 * 32 + r % 32 : r) * pitch + piece[q];
    }
  }
  FLA_DEVICE void copy(int q, char* lds, const MatSource* from, int wave) const {
    const MatSource& s = from[PAIR ? (wave * kCopies + q) / 4 & 1 : 0];
    mat_copy(s.descriptor(), piece[q] < s.left ? at[q] : kMatBeyond, lds + (wave * kCopies + q) * 1024);
  }
  // rows r0 .. r0+31 of the tile as the instruction takes them, quarter h of the slice
  static FLA_DEVICE i32x4 fragment(const char* lds, int r0, int h, int lane) {
    const int r = lane & 31;
    return *(const i32x4*)(lds + (r0 + r) * kSliceBytes + (((2 * h + (lane >> 5)) ^ key(r)) * 16));
  }
};

template <int ROWS>
struct Operand<ROWS, true, false> {
  static constexpr int kSources = 1, kBytes = ROWS * kSliceBytes, kCopies = ROWS / 32, kPieces = ROWS / 8, kDeep = 64 / kPieces;   // kDeep: k of a copy
  static FLA_DEVICE int key(int k) { return ROWS > 64 ? k & 3 : k >> 1 & 1; }
  uint32_t at[kCopies];
  FLA_DEVICE void start(int wave, int lane, uint32_t pitch) {
#pragma unroll
    for (int q = 0; q < kCopies; ++q) {
      const int k = (wave * kCopies + q) * kDeep + lane / kPieces;
      at[q] = (uint32_t)k * pitch + ((lane % kPieces) ^ key(k) << 2) * 16;
    }
  }
  FLA_DEVICE void copy(int q, char* lds, const MatSource* from, int wave) const { mat_copy(from->descriptor(), at[q], lds + (wave * kCopies + q) * 1024); }
  static FLA_DEVICE i32x4 fragment(const char* lds, int r0, int h, int lane) {
    const int j = lane & 15, k = 16 * h + 8 * (lane >> 5) + (j >> 2);
    const char* p = lds + k * ROWS * 2 + ((r0 >> 5) ^ key(k)) * 64 + (lane >> 4 & 1) * 32 + (j & 3) * 8;
    const i32x2 lo = __builtin_bit_cast(i32x2, lds_read_tr((lds_s16x4*)p));
    const i32x2 hi = __builtin_bit_cast(i32x2, lds_read_tr((lds_s16x4*)(p + 4 * ROWS * 2)));   // (the same key)
    return i32x4{lo[0], lo[1], hi[0], hi[1]};
  }
};

// The sums of a tile.  Lane l of wave (wm, wn) holds in acc[i][j][r] the sum of m = wm BM/2 + 32 i + l % 32 and n = wn BN/2 + 32 j + 8 (r / 4) + 4 (l / 32) + r % 4.
template <typename T, int BM, int BN, int RING, bool SM, bool SN, bool PAIR = false>
struct MatTile {
  static constexpr int MT = BM / 64, NT = BN / 64, kPiece = (BM + BN) * kSliceBytes, kLds = RING * kPiece;
  typedef Operand<BM, SM> OpM;
  typedef Operand<BN, SN, PAIR> OpN;
  typedef typename Mat<T>::acc acc_t;
  struct Frags {
    i32x4 m[MT][2], n[NT][2];
  };
  static constexpr int kCopies = OpM::kCopies + OpN::kCopies;

  OpM om;
  OpN on;
  int lane, wave, wm, wn;
  FLA_DEVICE void start(uint32_t pitch_m, uint32_t pitch_n) {
    lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 1, wn = wave & 1;
    om.start(wave, lane, pitch_m);
    on.start(wave, lane, pitch_n);
  }
  struct Slice {
    MatSource m[1], n[OpN::kSources];
    char* lds;
  };
  // `source(s, m, n)`: where slice s lies (n: an array of OpN::kSources); asked for slices behind the last one too, of which nothing may be left, or what
  // may be read (they are copied and not multiplied).
  template <typename F>
  static FLA_DEVICE Slice slice(char* lds, const F& source, int s, int piece) {
    Slice c;
    source(s, c.m, c.n);
    c.lds = lds + piece * kPiece;
    return c;
  }
  FLA_DEVICE void copy(const Slice& c, int q) const {
    if (q < OpM::kCopies) om.copy(q, c.lds, c.m, wave);
    else on.copy(q - OpM::kCopies, c.lds + OpM::kBytes, c.n, wave);
  }
  // The first slices are on their way; nobody reads LDS.
  template <typename F>
  FLA_DEVICE void begin(char* lds, int first, const F& source) const {
#pragma unroll
    for (int d = 0; d < RING; ++d) {
      const Slice c = slice(lds, source, first + d, d);
#pragma unroll
      for (int q = 0; q < kCopies; ++q) copy(c, q);
    }
  }
  // Slices first .. last - 1, at least one, behind begin().  LATER, five times LATER: with `later` 1 and 2 so many memory operations of this wave were
  // issued behind it (the stores of the tile before, which need not be waited for).
  template <int LATER, typename F>
  FLA_DEVICE void multiply(char* lds, int first, int last, int later, const F& source, acc_t (&acc)[MT][NT]) const {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] = acc_t{};
    constexpr int kFrags = 2 * (MT + NT), kProducts = 2 * MT * NT;
    auto read = [&](Frags& f, const char* from, int half, int q) {   // (in the order in which they are multiplied)
      const int h = q / (MT + NT), g = q % (MT + NT);
      if (g < NT) f.n[g][h] = OpN::fragment(from + OpM::kBytes, (wn * NT + g) * 32, 2 * half + h, lane);
      else f.m[g - NT][h] = OpM::fragment(from, (wm * MT + g - NT) * 32, 2 * half + h, lane);
    };
    // The products of half a slice, between them the reads of the next half and, with COPIES, the copies of a slice.  The order of the instructions is
    // kept: both go in the first three quarters of the products (copies in the first half 2 % slower, over the whole slice 10 %: they arrive late).
    auto half = [&](const Frags& now, Frags& next, const char* from, int which, const Slice& c, bool copies) {
      constexpr int r = kProducts * 3 / 4 > 0 ? kProducts * 3 / 4 : 1;
#pragma unroll
      for (int g = 0; g < kProducts; ++g) {
        const int h = g / (MT * NT), i = g / NT % MT, j = g % NT;
        acc[i][j] = Mat<T>::mma(now.n[j][h], now.m[i][h], acc[i][j]);
        if (g < r) {
#pragma unroll
          for (int q = g * kFrags / r; q < (g + 1) * kFrags / r; ++q) read(next, from, which, q);
          if (copies)
#pragma unroll
            for (int q = g * kCopies / r; q < (g + 1) * kCopies / r; ++q) copy(c, q);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    constexpr int kNewer = (RING - 1) * kCopies;
    constexpr auto most = [](int n) { return n < 63 ? n : 63; };   // (the counter's largest value)
    if (later == 2) asm volatile("s_waitcnt vmcnt(%0)" ::"i"(most(kNewer + 5 * LATER)) : "memory");
    else if (later) asm volatile("s_waitcnt vmcnt(%0)" ::"i"(most(kNewer + LATER)) : "memory");
    else asm volatile("s_waitcnt vmcnt(%0)" ::"i"(kNewer) : "memory");
    asm volatile("s_barrier" ::: "memory");
    Frags f[2];
#pragma unroll
    for (int q = 0; q < kFrags; ++q) read(f[0], lds, 0, q);
    int piece = 0;   // of slice s
    Slice c;
    for (int s = first; s < last; ++s) {
      half(f[0], f[1], lds + piece * kPiece, 1, c, false);
      // this wave's copies of slice s + 1 have arrived and its fragments of s are read; then everybody's
      if (later == 2 && s == first) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"i"(most((RING - 2) * kCopies + 5 * LATER)) : "memory");
      else if (later && s == first) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"i"(most((RING - 2) * kCopies + LATER)) : "memory");
      else asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"i"((RING - 2) * kCopies) : "memory");
      asm volatile("s_barrier" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      c = slice(lds, source, s + RING, piece);
      piece = piece + 1 < RING ? piece + 1 : 0;
      half(f[1], f[0], lds + piece * kPiece, 0, c, true);
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");   // no copy into LDS outlives the tile
  }
};

// Neighbouring workgroup numbers go to different XCDs: each XCD takes a run of `total` tiles
FLA_DEVICE uint32_t mat_turn(uint32_t block, uint32_t total) {
  const uint32_t xcd = block % 8, per = total / 8, rest = total % 8;
  return xcd * per + (xcd < rest ? xcd : rest) + block / 8;
}
// Tile number `id`: eight rows of tiles deep, so that those side by side share operands in an L2
FLA_DEVICE void mat_place(uint32_t id, uint32_t tm_all, uint32_t tn_all, uint32_t* tm, uint32_t* tn) {
  const uint32_t deep = tm_all < 8 ? tm_all : 8, band = id / (deep * tn_all), in = id - band * deep * tn_all;
  const uint32_t rows_in = tm_all - band * deep < deep ? tm_all - band * deep : deep, col = in / rows_in;
  *tm = band * deep + in - col * rows_in, *tn = col;
}

// The tiles of a launch of one workgroup a CU: `whole` of them by workgroups in turn, and, where the rest would leave half of the CUs or more without
// one, the rest as `halves` tiles of half the columns.
struct MatGrid {
  uint32_t tm, tn, whole, halves;
};
// A workgroup's tiles, one behind the other.  The first copies of a tile are on their way while the sums of the one before are brought out: what is waited for
// between two tiles is a barrier.  Half of the workgroups take their half tile first: then not all of them write at the same time.  JOB:
//   Whole, Half        MatTile types;  LATER  memory operations of a wave that finish() of a whole tile issues where it returns 1, a fifth of those where it returns 2
//   at(tm, n)          remembers where the tile lies: row of tiles tm, first column n (in units of half tiles)
//   columns(side)      sends what goes by row and column into LDS, half `side` of it (a load in finish() would wait for the copies ahead of it);   source(s, m, n)   as for MatTile
//   finish(tile, acc, side)   brings a tile out
template <typename Job>
FLA_DEVICE void mat_run(char* lds, const MatGrid& grid, Job& job) {
  typedef typename Job::Whole Whole;
  typedef typename Job::Half Half;
  auto source = [&](int s, MatSource* m, MatSource* n) { job.source(s, m, n); };
  int side = 0;
  const bool early = blockIdx.x / 8 % 2;      // (every second one of an XCD's)
#pragma unroll 1
  for (int turn = 0; turn < 2; ++turn) {
    if (Job::kHalves && early == (turn == 0)) {
      if (blockIdx.x >= grid.halves) continue;
      Half tile;
      job.start(tile);
      const uint32_t id = mat_turn(blockIdx.x, grid.halves);
      uint32_t tm, tn;
      mat_place(grid.whole + id / 2, grid.tm, grid.tn, &tm, &tn);
      __syncthreads();
      job.at(tm, tn * 2 + id % 2);
      job.columns(side);
      tile.begin(lds, job.first, source);
      typename Half::acc_t acc[Half::MT][Half::NT];
      tile.template multiply<0>(lds, job.first, job.last, 0, source, acc);
      job.finish(tile, acc, side);
      side ^= 1;
    } else if (!Job::kHalves && turn) {
      break;
    } else {
      Whole whole;
      job.start(whole);
      uint32_t u = blockIdx.x;
      auto begin = [&](uint32_t id) {
        uint32_t tm, tn;
        mat_place(id, grid.tm, grid.tn, &tm, &tn);
        job.at(tm, tn * 2);
        job.columns(side);
        whole.begin(lds, job.first, source);
      };
      if (u >= grid.whole) continue;
      __syncthreads();
      begin(mat_turn(u, grid.whole));
      int later = 0;
      for (;;) {
        typename Whole::acc_t acc[Whole::MT][Whole::NT];
        whole.template multiply<Job::LATER>(lds, job.first, job.last, later, source, acc);
        u += gridDim.x;
        const bool more = u < grid.whole;
        const Job done = job;
        const int now = side;
        side ^= 1;
        if (more) {
          asm volatile("s_barrier" ::: "memory");   // nobody reads the slices any more
          begin(mat_turn(u, grid.whole));
        }
        later = done.finish(whole, acc, now);
        if (!more) break;
      }
    }
  }
}

// Between the pieces of a tile that are brought out: without it the compiler brings the operands of all of them into registers first
FLA_DEVICE void mat_piece_end() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// The sums of 32 x 32 elements as they are brought out.  Those of a tile that has all the accumulation registers stay there until then: left to itself the
// compiler moves all 256 into ordinary registers at the loop's end and spills what lives on.
template <typename Tile>
FLA_DEVICE typename Tile::acc_t mat_sums(const typename Tile::acc_t (&acc)[Tile::MT][Tile::NT], int i, int j) {
  typename Tile::acc_t v = acc[i][j];
  if constexpr (Tile::MT * Tile::NT == 16) asm volatile("" : "+a"(v));
  return v;
}

// Eight consecutive n a lane from two runs of four, packed in pairs (a, b: the lane's of r / 4 even and of the odd one behind it): lane l then holds
// those from 8 (r / 4 + l / 32) on.
FLA_DEVICE i32x4 mat_join(u32x2 a, u32x2 b) {
  const u32x2 p = __builtin_amdgcn_permlane32_swap(a[0], b[0], false, false), q = __builtin_amdgcn_permlane32_swap(a[1], b[1], false, false);
  return i32x4{(int)p[0], (int)q[0], (int)p[1], (int)q[1]};
}

// Eight consecutive elements (of 16 bits) of a row from n on, of which those below N exist, at any element address
template <typename O>
FLA_DEVICE void store_piece(O* row, int64_t n, int64_t N, i32x4 v) {
  typedef i32x4 any __attribute__((aligned(2)));
  if (n + 8 <= N) {
    *(any*)(row + n) = v;
  } else {   // (a loop: unrolled, the pieces of a tile are a hundred thousand bytes of code)
    uint16_t* to = (uint16_t*)(row + n);
    const int count = (int)(N - n);
#pragma unroll 1
    for (int i = 0; i < count; ++i) {
      to[i] = (uint16_t)v[0];
      v[0] = __builtin_amdgcn_alignbit(v[1], v[0], 16), v[1] = __builtin_amdgcn_alignbit(v[2], v[1], 16);
      v[2] = __builtin_amdgcn_alignbit(v[3], v[2], 16), v[3] = (int)((uint32_t)v[3] >> 16);
    }
  }
}
template <typename O>
FLA_DEVICE u32x2 pack4(const float* v) {
  typename Elem<O>::v4 e;
#pragma unroll
  for (int i = 0; i < 4; ++i) e[i] = (O)v[i];
  return __builtin_bit_cast(u32x2, e);
}

}  // namespace
