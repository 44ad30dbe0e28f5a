// The elementwise gated recurrence h_t = a_t h_{t-1} + u_t, what its forward and backward launches share.
//
// A step is an affine map of the state, so a run of steps is one too: (A, H) with h -> A h + H, joined in order.  A workgroup
// owns 64 channels of a segment of a sequence and goes through it in tiles: eight waves of 8 R rows, a lane R = 2 or 4 rows of eight
// channels (16 bytes a load in 16 bits, a wave's load covers eight whole 128-byte rows).  A tile is joined in
// three levels: the lane's rows in registers, the eight row groups of a wave by shuffles, the waves through LDS (one
// barrier a tile).  Between tiles the state stays in a register of the lane with that channel's number.  Rows past the end of a segment are
// read as steps that change nothing: a log decay of 0, a forget gate of plus infinity, an input and a gradient of 0.
//
// Bounds and figures (bf16, us): 8 x 4096 x 2048 runs uncut, one workgroup a CU.  Log decays in fp32, forward: 114, 4.7 TB/s.  From pre-activations
// with a lower bound: forward 95 - 105 with the states for the backward (4.0 - 4.4 TB/s), backward 169 - 204 (3.4 - 4.1 TB/s; the vector units are busy for
// two thirds of it, 51 instructions an element, the rest is latency that two waves a SIMD do not cover).  With gates in fp32 119 and 215, all in
// fp32 171 and 305: 1.1 times the time of a copy of as many bytes.  32 channels to a workgroup, which leave half of every
// 128-byte line to another one: forward 135 instead of 117; sixteen waves of half the rows: 121.
//
// Sequences are cut into segments where (sequence, 64 channels) pairs would leave CUs idle; a first launch then forms each
// segment's map, and every workgroup of the second joins the maps of the segments ahead of its own (a fixed order, no atomics,
// nothing waits for another workgroup).  One prompt of 8191 x 2048: 19.4 for the maps, which read both operands once more, and 28.8.
#pragma once
#include "fla_common.h"
#include "row_vec.h"

namespace {

constexpr int kCh = 64;                           // channels of a workgroup
constexpr int kWaves = 8, kGroups = 8;            // waves of a workgroup, row groups of a wave
constexpr int kKept = FLA_HGRN_STATE_ROWS;        // rows from one kept state to the next
static_assert(kKept == kGroups * 2, "a wave of the backward (R = 2) starts from a kept state");
static_assert(FLA_HGRN_TILE == kWaves * kGroups * 4, "a segment is whole tiles of either kind");
// what the operands hold
enum Gates { kLogDecays = 0, kGates = 1, kBoundedGates = 2 };

struct HgrnParams {
  const void* x;        // u, or the pre-activations i  [B,T,D], rows ldx apart
  const void* g;        // log a, or the pre-activations f, rows ldg apart
  const float* lb;      // [D] or NULL
  const float* h0;      // [N,D] or NULL
  void* o;              // [B,T,D]
  float* ht;            // [N,D] or NULL
  float* states;        // [B*T / 16 + N + 1, D] or NULL: the state ahead of every 16 rows of a sequence
  float* maps;          // [segments, 2, D] or NULL (uncut)
  // backward
  const void* dout;     // [B,T,D] or NULL (zeros)
  const float* dht;     // [N,D] or NULL (zeros)
  void* dx;
  void* dg;
  float* dh0;           // [N,D] or NULL
  float* dlb;           // [segments, D] or NULL
  const int64_t* offsets;
  const int64_t* indices;       // [NT,2] (sequence, segment)
  const int64_t* chunk_offsets; // [N+1] first segment of a sequence
  int64_t NT, segment, T, ldx, ldg;
  int D, ncb, nseg;     // nseg: segments of a sequence of a batch without offsets
};

struct Segment {
  int64_t n, c, count, first;   // sequence, number in it, segments of it, its first one
  int64_t bos, begin, len;      // rows: the sequence's first, the segment's first, the segment's number
  int64_t id;                   // n's segment c among all
};
// Segment number `id`; of a packed batch's numbers from NT on, NT + n stands for sequence n if that is empty.
FLA_DEVICE Segment find_segment(const HgrnParams& p, int64_t id, bool* exists) {
  Segment s;
  s.id = id;
  *exists = true;
  if (!p.offsets) {
    s.n = id / p.nseg;
    s.c = id % p.nseg;
    s.count = p.nseg;
    s.first = s.n * p.nseg;
    s.bos = s.n * p.T;
    s.begin = s.bos + s.c * p.segment;
    s.len = p.T - s.c * p.segment;
  } else if (id < p.NT) {
    s.n = p.indices[2 * id];
    s.c = p.indices[2 * id + 1];
    s.first = p.chunk_offsets[s.n];
    s.count = p.chunk_offsets[s.n + 1] - s.first;
    s.bos = p.offsets[s.n];
    s.begin = s.bos + s.c * p.segment;
    s.len = p.offsets[s.n + 1] - s.begin;
  } else {
    s.n = id - p.NT;
    s.c = 0;
    s.first = 0;
    s.count = 1;
    s.bos = s.begin = p.offsets[s.n];
    s.len = 0;
    *exists = p.offsets[s.n + 1] == s.bos;
  }
  if (s.len > p.segment) s.len = p.segment;
  return s;
}
// The kept states of sequence n, which begins at row bos, start here: no two sequences share a slot.
FLA_DEVICE int64_t state_slot(const Segment& s) { return s.bos / kKept + s.n; }

// sigmoid(x) and 1 - sigmoid(x), each to its own relative precision: from e^{-|x|}, which neither overflows nor cancels
FLA_DEVICE void sigmoid_both(float x, float* s, float* rest) {
  const float z = __expf(-__builtin_fabsf(x)), r = __builtin_amdgcn_rcpf(1.f + z), small = z * r;
  *s = x >= 0.f ? r : small;
  *rest = x >= 0.f ? small : r;
}

// Element offset of the lane's piece of its first row within the wave's rows; rows of at most 2^24 elements keep it in 32 bits
template <int R>
FLA_DEVICE uint32_t lane_at(int lane, int64_t ld) { return (uint32_t)(lane >> 3) * R * (uint32_t)ld + (lane & 7) * VEC; }

template <bool V>
struct Full {
  static constexpr bool value = V;
};
// The lane's rows of a tile: `rows` is the wave's first row (64 channels from `cb` on), of which `left` exist.  FULL: all of the wave's rows and
// channels exist, and no branch stands around the loads: the compiler counts what is in flight behind a load, and where a branch may have
// skipped some of it, waits for all of it instead, the stores of the tile before included.
template <typename T, bool WIDE, int R, bool FULL>
FLA_DEVICE void fetch_rows(typename Row8<T>::raw (&r)[R], const T* rows, int64_t ld, uint32_t at, int64_t left, int group, int valid, float fill) {
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (FULL) r[i] = Row8<T>::load_raw(rows + i * ld + at);
    else r[i] = load_raw8<T, WIDE>(rows + i * ld + at, group * R + i < left ? valid : 0, fill);
  }
}
template <typename T, bool WIDE, int R, bool FULL>
FLA_DEVICE void store_row(T* rows, int64_t ld, uint32_t at, int i, const float* v, int64_t left, int group, int valid) {
  if (FULL) Row8<T>::store(rows + i * ld + at, v);
  else store8<T, WIDE>(rows + i * ld + at, v, group * R + i < left ? valid : 0);
}

// A map on its way through the eight row groups of a wave: joined with those of lower (UP) or higher groups, own group included
template <bool UP>
FLA_DEVICE void join_groups(float A[VEC], float H[VEC], int group) {
#pragma unroll
  for (int d = 1; d < kGroups; d *= 2) {
    const bool has = UP ? group >= d : group + d < kGroups;
    float a[VEC], h[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      a[i] = UP ? __shfl_up(A[i], 8 * d, 64) : __shfl_down(A[i], 8 * d, 64);
      h[i] = UP ? __shfl_up(H[i], 8 * d, 64) : __shfl_down(H[i], 8 * d, 64);
    }
    if (has) {   // (a branch: selects would cost as much as the arithmetic)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        H[i] = fmaf(A[i], h[i], H[i]);
        A[i] *= a[i];
      }
    }
  }
}

// What the waves of a tile exchange: their maps (two tiles' worth: one barrier a tile), and a wave's own entering state.
struct TileShare {
  float A[2][kWaves][kCh], H[2][kWaves][kCh];
  float in[kWaves][kCh];
  float lb[kCh];       // the lower bounds: read again for every tile, eight registers less
};
// The lower bounds of the workgroup's channels into LDS (channels that are not there: 0)
FLA_DEVICE void keep_bounds(TileShare& sh, const float* lb, int first, int D) {
  if (threadIdx.x < kCh) sh.lb[threadIdx.x] = first + (int)threadIdx.x < D ? lb[first + threadIdx.x] : 0.f;
  __syncthreads();
}
FLA_DEVICE void bounds_of(const TileShare& sh, int lane, float o[VEC]) {
  const int c = (lane & 7) * VEC;
  const f32x4 a = *(const f32x4*)&sh.lb[c], b = *(const f32x4*)&sh.lb[c + 4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    o[i] = a[i];
    o[4 + i] = b[i];
  }
}
// Leaves a wave's map, whose eight channels the lanes of one group hold, and returns the state that enters this wave; `carry`,
// the state that enters the tile, becomes the one that leaves it (both for the channel with the lane's number), and `all` the
// product of the decays.  UP: waves in ascending order.
template <bool UP>
FLA_DEVICE float join_waves(TileShare& sh, int buf, const float A[VEC], const float H[VEC], bool holds, int wave, int lane,
                            float* carry, float* all) {
  if (holds) {
    const int c = (lane & 7) * VEC;
    *(f32x4*)&sh.A[buf][wave][c] = f32x4{A[0], A[1], A[2], A[3]};
    *(f32x4*)&sh.A[buf][wave][c + 4] = f32x4{A[4], A[5], A[6], A[7]};
    *(f32x4*)&sh.H[buf][wave][c] = f32x4{H[0], H[1], H[2], H[3]};
    *(f32x4*)&sh.H[buf][wave][c + 4] = f32x4{H[4], H[5], H[6], H[7]};
  }
  lds_barrier();
  float c = *carry, mine = c, prod = *all;
#pragma unroll 4
  for (int k = 0; k < kWaves; ++k) {
    const int w = UP ? k : kWaves - 1 - k;
    if (w == wave) mine = c;
    const float a = sh.A[buf][w][lane];
    c = fmaf(a, c, sh.H[buf][w][lane]);
    prod *= a;
  }
  *carry = c;
  *all = prod;
  return mine;
}
// The lane's eight channels of a value that lanes hold by channel number (within the wave: LDS operations of one wave are in order)
FLA_DEVICE void spread(TileShare& sh, float v, int wave, int lane, float o[VEC]) {
  sh.in[wave][lane] = v;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  const int c = (lane & 7) * VEC;
  const f32x4 a = *(const f32x4*)&sh.in[wave][c], b = *(const f32x4*)&sh.in[wave][c + 4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    o[i] = a[i];
    o[4 + i] = b[i];
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}
// joins the map of a run of steps onto the state ahead of it
FLA_DEVICE float onto(float A, float H, float h) { return fmaf(A, h, H); }

// the types of (x, g)
#define HGRN_TYPES(D) \
  D(FLA_BF16, bf16, FLA_BF16, bf16) D(FLA_BF16, bf16, FLA_F32, float) D(FLA_F16, f16, FLA_F16, f16) \
  D(FLA_F16, f16, FLA_F32, float) D(FLA_F32, float, FLA_F32, float)

constexpr int64_t kMostWorkgroups = 0xffffffff / (kWaves * 64);   // (a launch is less than 2^32 threads)
// whether rows ld apart can be read 16 bytes at a time
inline bool wide_rows(const void* p, int64_t ld, int64_t D, int type) {
  const int64_t e = type == FLA_F32 ? 4 : 2;
  return (uintptr_t)p % 16 == 0 && ld * e % 16 == 0 && D % VEC == 0;
}

}  // namespace
