// Forward of the elementwise gated recurrence h_t = a_t h_{t-1} + u_t, o = h (see hgrn_scan.h for the scan), and its single step.
#include "hgrn_scan.h"

namespace {

// OUT: writes o (and ht, states); otherwise the map of the segment.  R = 4 rows a lane in long whole sequences, R = 2 in cut and short ones, whose
// workgroups share CUs (107 registers instead of 161 - 203).  Whole tiles have no branch around their loads and stores: a
// training step of 8 x 4096 x 2048 takes 262 us instead of 312.
template <typename T, typename GT, int GATES, bool WIDE, bool OUT, int R>
__global__ __launch_bounds__(kWaves * 64) void hgrn_fwd_kernel(HgrnParams p) {
  constexpr int kSpan = kGroups * R, kTile = kWaves * kSpan;   // rows of a wave, of the workgroup
  __shared__ __attribute__((aligned(16))) TileShare sh;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = lane >> 3;
  const int cb = blockIdx.x % p.ncb, D = p.D;
  bool exists;
  const Segment s = find_segment(p, blockIdx.x / p.ncb, &exists);
  if (!exists) return;
  if (!OUT && s.c + 1 == s.count) return;     // nothing follows the last segment of a sequence
  const int ch = cb * kCh + lane;             // the channel this lane carries between tiles
  const int col = cb * kCh + (lane & 7) * VEC, valid = D - col;   // the eight it scans
  if (GATES == kBoundedGates) keep_bounds(sh, p.lb, cb * kCh, D);

  // the wave's rows of the tile that is fetched
  const int64_t row0 = s.begin + wave * kSpan;
  const T* xr = (const T*)p.x + row0 * p.ldx + cb * kCh;
  const GT* gr = (const GT*)p.g + row0 * p.ldg + cb * kCh;
  T* orow = (T*)p.o + row0 * D + cb * kCh;
  const uint32_t ax = lane_at<R>(lane, p.ldx), ag = lane_at<R>(lane, p.ldg), ao = lane_at<R>(lane, D);
  const int64_t left = s.len - wave * kSpan;
  typename Row8<T>::raw nx[R];
  typename Row8<GT>::raw ng[R];
  auto fetch = [&](int64_t t0, auto full) {
    constexpr bool F = decltype(full)::value;
    fetch_rows<T, WIDE, R, F>(nx, xr + t0 * p.ldx, p.ldx, ax, left - t0, group, valid, 0.f);
    fetch_rows<GT, WIDE, R, F>(ng, gr + t0 * p.ldg, p.ldg, ag, left - t0, group, valid, GATES ? __builtin_inff() : 0.f);
  };
  // tiles of which all rows and channels exist
  const int64_t whole = WIDE && cb * kCh + kCh <= D ? s.len / kTile * kTile : 0;
  if (whole > 0) fetch(0, Full<true>());
  else fetch(0, Full<false>());
  float carry = 0.f, all = 1.f;
  if (OUT && ch < D) {
    if (p.h0) carry = p.h0[s.n * D + ch];
    const float* m = p.maps + s.first * 2 * D + ch;
#pragma unroll 4
    for (int64_t k = 0; k < s.c; ++k) carry = onto(m[2 * k * D], m[(2 * k + 1) * D], carry);
  }
  int buf = 0;
  auto tile = [&](int64_t t0, auto full, auto full_next) {
    float a[R][VEC], u[R][VEC], A[VEC], H[VEC];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      Row8<T>::unpack(nx[r], u[r]);
      Row8<GT>::unpack(ng[r], a[r]);
    }
    fetch(t0 + kTile, full_next);
    float lb[VEC];
    if (GATES == kBoundedGates) bounds_of(sh, lane, lb);
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        if (GATES) {
          float sf, rest;
          sigmoid_both(a[r][i], &sf, &rest);
          u[r][i] = u[r][i] * sigmoidf(u[r][i]);
          if (GATES == kBoundedGates) {
            u[r][i] *= (1.f - lb[i]) * rest;
            a[r][i] = fmaf(1.f - lb[i], sf, lb[i]);
          } else {
            u[r][i] *= rest;
            a[r][i] = sf;
          }
        } else {
          a[r][i] = __expf(a[r][i]);
        }
        H[i] = r ? fmaf(a[r][i], H[i], u[r][i]) : u[r][i];
        A[i] = r ? A[i] * a[r][i] : a[r][i];
      }
    }
    join_groups<true>(A, H, group);
    const float mine = join_waves<true>(sh, buf, A, H, group == kGroups - 1, wave, lane, &carry, &all);
    buf ^= 1;
    if (!OUT) return;
    const int64_t n = left - t0;
    if (!decltype(full)::value && n <= 0) return;   // (uniform, and no barrier behind it)
    float h[VEC];
    spread(sh, mine, wave, lane, h);
    // the state behind the groups ahead: that of the neighbour's last row
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float before = __shfl_up(onto(A[i], H[i], h[i]), 8, 64);
      h[i] = group > 0 ? before : h[i];
    }
    if (p.states && group * R % kKept == 0) {
      const int t = group * R;
      store8<float, WIDE>(p.states + (state_slot(s) + (s.c * p.segment + t0 + wave * kSpan + t) / kKept) * D + col, h, t < n ? valid : 0);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) h[i] = fmaf(a[r][i], h[i], u[r][i]);
      store_row<T, WIDE, R, decltype(full)::value>(orow + t0 * D, D, ao, r, h, n, group, valid);
    }
  };
  int64_t t0 = 0;
  for (; t0 + kTile < whole; t0 += kTile) tile(t0, Full<true>(), Full<true>());
  if (t0 < whole) tile(t0, Full<true>(), Full<false>()), t0 += kTile;
  for (; t0 < s.len; t0 += kTile) tile(t0, Full<false>(), Full<false>());
  if (wave == 0 && ch < D) {
    if (!OUT) {
      float* m = p.maps + s.id * 2 * D + ch;
      m[0] = all;
      m[D] = carry;
    } else if (p.ht && s.c + 1 == s.count) {
      p.ht[s.n * D + ch] = carry;
    }
  }
}

struct StepParams {
  const void* x;
  const void* g;
  const float* lb;
  const float* h0;
  void* o;
  float* ht;
  int64_t N, ldx, ldg;
  int D;
};
// One token per sequence, a lane eight channels.  Latency: a step of 32 sequences of 2048 channels moves 0.9 MB.
template <typename T, typename GT, int GATES, bool WIDE>
__global__ __launch_bounds__(64) void hgrn_step_kernel(StepParams p) {
  const int per = (p.D + VEC - 1) / VEC;
  const int64_t id = (int64_t)blockIdx.x * 64 + threadIdx.x, n = id / per;
  if (n >= p.N) return;
  const int col = (int)(id % per) * VEC, valid = p.D - col;
  float u[VEC], a[VEC], h[VEC];
  const auto rx = load_raw8<T, WIDE>((const T*)p.x + n * p.ldx + col, valid);
  const auto rg = load_raw8<GT, WIDE>((const GT*)p.g + n * p.ldg + col, valid);
  float lb[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    h[i] = p.h0 && i < valid ? p.h0[n * p.D + col + i] : 0.f;
    lb[i] = GATES == kBoundedGates && i < valid ? p.lb[col + i] : 0.f;
  }
  Row8<T>::unpack(rx, u);
  Row8<GT>::unpack(rg, a);
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    if (GATES) {
      float sf, rest;
      sigmoid_both(a[i], &sf, &rest);
      h[i] = fmaf(fmaf(1.f - lb[i], sf, lb[i]), h[i], (1.f - lb[i]) * rest * (u[i] * sigmoidf(u[i])));
    } else {
      h[i] = fmaf(__expf(a[i]), h[i], u[i]);
    }
  }
  store8<T, WIDE>((T*)p.o + n * p.D + col, h, valid);
  if (p.ht) {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (i < valid) p.ht[n * p.D + col + i] = h[i];
  }
}

template <typename T, typename GT, int GATES, bool WIDE>
int launch_fwd(const HgrnParams& p, int64_t segments, int64_t empty, hipStream_t st) {
  if (p.maps) {
    hipLaunchKernelGGL((hgrn_fwd_kernel<T, GT, GATES, WIDE, false, 2>), dim3((unsigned)(segments * p.ncb)), dim3(kWaves * 64), 0, st, p);
    FLA_CHECK_LAUNCH();
    hipLaunchKernelGGL((hgrn_fwd_kernel<T, GT, GATES, WIDE, true, 2>), dim3((unsigned)((segments + empty) * p.ncb)), dim3(kWaves * 64), 0, st, p);
    FLA_CHECK_LAUNCH();
    return FLA_OK;
  }
  // Uncut.  Short sequences leave less of a tile of 128 rows empty than of one of 256, and two workgroups share a CU if there are that many (us, 2048
  // channels, R = 2 and 4): 256 x 128 tokens 96 and 185, 64 x 300 58 and 89, 64 x 512 87 and 97; 6 x 4096 87 and 77, 16 x 2048 102 and 96.
  const int64_t grid = (segments + empty) * p.ncb;
  if (p.segment <= 1024 && grid > 256)
    hipLaunchKernelGGL((hgrn_fwd_kernel<T, GT, GATES, WIDE, true, 2>), dim3((unsigned)grid), dim3(kWaves * 64), 0, st, p);
  else
    hipLaunchKernelGGL((hgrn_fwd_kernel<T, GT, GATES, WIDE, true, 4>), dim3((unsigned)grid), dim3(kWaves * 64), 0, st, p);
  FLA_CHECK_LAUNCH();
  return FLA_OK;
}

template <typename T, typename GT, int GATES, bool WIDE>
int launch_step(const StepParams& p, hipStream_t st) {
  hipLaunchKernelGGL((hgrn_step_kernel<T, GT, GATES, WIDE>), dim3((unsigned)fla_cdiv(p.N * fla_cdiv(p.D, VEC), 64)), dim3(64), 0, st, p);
  FLA_CHECK_LAUNCH();
  return FLA_OK;
}

}  // namespace

extern "C" int64_t fla_hgrn_segment(int64_t n_seqs, int64_t tokens, int64_t longest, int64_t D) {
  if (n_seqs <= 0 || tokens <= 0 || longest <= 0 || D <= 0) return FLA_HGRN_TILE;
  const int64_t cbs = fla_cdiv(D, kCh), whole = fla_cdiv(longest, FLA_HGRN_TILE) * FLA_HGRN_TILE;
  // Whole sequences where all of them are as much work as 144 chains of the longest side by side (us forward / backward, 4096 tokens of 2048 channels, whole
  // and cut: 4 sequences, 128 chains, 70 / 147 and 79 / 125; 5: 69 / 149 and 105 / 161); otherwise four workgroups a CU, at most 64 segments to a
  // sequence (a workgroup joins the maps of all segments ahead of its own).  8191 tokens of 2048 channels: 47 us from 512 workgroups on,
  // 55 with 256; 12 sequences of 16384 tokens in all, 1000 channels, both ways: 151, 144, 144 us with 512, 1024, 2048.
  if (tokens * cbs >= 144 * longest) return whole;
  int64_t seg = fla_cdiv(fla_cdiv(tokens * cbs, 1024), FLA_HGRN_TILE) * FLA_HGRN_TILE;
  const int64_t least = fla_cdiv(fla_cdiv(longest, 64), FLA_HGRN_TILE) * FLA_HGRN_TILE;
  if (seg < least) seg = least;
  return seg < whole ? seg : whole;
}

extern "C" int fla_hgrn_fwd(const void* x, const void* g, const float* lower_bound, const float* h0, void* o, float* ht, float* states,
                            float* maps, const int64_t* offsets, const int64_t* indices, const int64_t* chunk_offsets, int64_t NT,
                            int64_t segment, int gates, int x_dtype, int g_dtype, int64_t B, int64_t T, int64_t D, int64_t N,
                            int64_t ldx, int64_t ldg, fla_stream_t stream) {
  FLA_REQUIRE(x && g && o && B > 0 && T > 0 && D > 0 && N > 0 && NT >= 0 && ldx >= D && ldg >= D, FLA_E_INVALID);
  FLA_REQUIRE(segment > 0 && segment % FLA_HGRN_TILE == 0 && (!lower_bound || gates), FLA_E_INVALID);
  FLA_REQUIRE(offsets ? B == 1 && (indices || NT == 0) && chunk_offsets : N == B, FLA_E_INVALID);
  FLA_REQUIRE((uintptr_t)states % 16 == 0, FLA_E_ALIGNMENT);
  const int64_t nseg = fla_cdiv(T, segment), cbs = fla_cdiv(D, kCh), segments = offsets ? NT : B * nseg;
  FLA_REQUIRE(maps || offsets || nseg == 1, FLA_E_INVALID);
  FLA_REQUIRE(ldx <= FLA_HGRN_MAX_PITCH && ldg <= FLA_HGRN_MAX_PITCH && segments + N <= kMostWorkgroups / cbs, FLA_E_UNSUPPORTED);
  HgrnParams p{};
  p.x = x, p.g = g, p.lb = lower_bound, p.h0 = h0, p.o = o, p.ht = ht, p.states = states, p.maps = maps;
  p.offsets = offsets, p.indices = indices, p.chunk_offsets = chunk_offsets;
  p.NT = NT, p.segment = segment, p.T = T, p.ldx = ldx, p.ldg = ldg;
  p.D = (int)D, p.ncb = (int)cbs, p.nseg = (int)nseg;
  const bool wide = wide_rows(x, ldx, D, x_dtype) && wide_rows(g, ldg, D, g_dtype) && wide_rows(o, D, D, x_dtype);
  const int64_t empty = offsets ? N : 0;
  const int kind = !gates ? kLogDecays : lower_bound ? kBoundedGates : kGates;
  hipStream_t st = (hipStream_t)stream;
#define D_(XE, XT, GE, GT)                                                                                       \
  if (x_dtype == XE && g_dtype == GE) {                                                                          \
    if (kind == kLogDecays) return wide ? launch_fwd<XT, GT, 0, true>(p, segments, empty, st) : launch_fwd<XT, GT, 0, false>(p, segments, empty, st); \
    if (kind == kGates) return wide ? launch_fwd<XT, GT, 1, true>(p, segments, empty, st) : launch_fwd<XT, GT, 1, false>(p, segments, empty, st); \
    return wide ? launch_fwd<XT, GT, 2, true>(p, segments, empty, st) : launch_fwd<XT, GT, 2, false>(p, segments, empty, st); \
  }
  HGRN_TYPES(D_)
#undef D_
  return FLA_E_UNSUPPORTED;
}

extern "C" int fla_hgrn_step(const void* x, const void* g, const float* lower_bound, const float* h0, void* o, float* ht, int gates,
                             int x_dtype, int g_dtype, int64_t N, int64_t D, int64_t ldx, int64_t ldg, fla_stream_t stream) {
  FLA_REQUIRE(x && g && o && N > 0 && D > 0 && ldx >= D && ldg >= D && (!lower_bound || gates), FLA_E_INVALID);
  FLA_REQUIRE(ldx <= FLA_HGRN_MAX_PITCH && ldg <= FLA_HGRN_MAX_PITCH && N <= 0x7fffffff / fla_cdiv(D, VEC), FLA_E_UNSUPPORTED);
  const StepParams p{x, g, lower_bound, h0, o, ht, N, ldx, ldg, (int)D};
  const bool wide = wide_rows(x, ldx, D, x_dtype) && wide_rows(g, ldg, D, g_dtype) && wide_rows(o, D, D, x_dtype);
  const int kind = !gates ? kLogDecays : lower_bound ? kBoundedGates : kGates;
  hipStream_t st = (hipStream_t)stream;
#define D_(XE, XT, GE, GT)                                                                                                   \
  if (x_dtype == XE && g_dtype == GE) {                                                                                      \
    if (kind == kLogDecays) return wide ? launch_step<XT, GT, 0, true>(p, st) : launch_step<XT, GT, 0, false>(p, st); \
    if (kind == kGates) return wide ? launch_step<XT, GT, 1, true>(p, st) : launch_step<XT, GT, 1, false>(p, st);     \
    return wide ? launch_step<XT, GT, 2, true>(p, st) : launch_step<XT, GT, 2, false>(p, st);                         \
  }
  HGRN_TYPES(D_)
#undef D_
  return FLA_E_UNSUPPORTED;
}
