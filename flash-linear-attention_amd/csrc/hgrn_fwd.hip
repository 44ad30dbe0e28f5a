// Forward of the elementwise gated recurrence h_t = a_t h_{t-1} + u_t, o = h (see hgrn_scan.h for the scan), and its single step.
#include "hgrn_scan.h"

namespace {

// OUT: writes o (and ht, states); otherwise the map of the segment.
template <typename T, typename GT, bool GATES, bool WIDE, bool OUT>
__global__ __launch_bounds__(kWaves * 64) void hgrn_fwd_kernel(HgrnParams p) {
  __shared__ __attribute__((aligned(16))) TileShare sh;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = lane >> 3;
  const int cb = blockIdx.x % p.ncb, D = p.D;
  bool exists;
  const Segment s = find_segment(p, blockIdx.x / p.ncb, &exists);
  if (!exists) return;
  const int ch = cb * kCh + lane;             // the channel this lane carries between tiles
  const int col = cb * kCh + (lane & 7) * VEC, valid = D - col;   // the eight it scans
  if (!OUT && s.c + 1 == s.count) return;     // nothing follows the last segment of a sequence
  float lb[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) lb[i] = GATES && p.lb && i < valid ? p.lb[col + i] : 0.f;

  constexpr int kRows = kFwdRows, kSpan = kGroups * kRows, kTile = kWaves * kSpan;
  typename Row8<T>::raw nx[kRows];
  typename Row8<GT>::raw ng[kRows];
  auto fetch = [&](int64_t t0) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int64_t t = t0 + wave * kSpan + group * kRows + r, row = s.begin + t;
      const int v = t < s.len ? valid : 0;
      nx[r] = load_raw8<T, WIDE>((const T*)p.x + row * p.ldx + col, v);
      ng[r] = load_raw8<GT, WIDE>((const GT*)p.g + row * p.ldg + col, v);
    }
  };
  fetch(0);
  float carry = 0.f, all = 1.f;
  if (OUT && ch < D) {
    if (p.h0) carry = p.h0[s.n * D + ch];
    const float* m = p.maps + s.first * 2 * D + ch;
#pragma unroll 8
    for (int64_t k = 0; k < s.c; ++k) carry = onto(m[2 * k * D], m[(2 * k + 1) * D], carry);
  }
  int buf = 0;
  for (int64_t t0 = 0; t0 < s.len; t0 += kTile, buf ^= 1) {
    float a[kRows][VEC], u[kRows][VEC];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      Row8<T>::unpack(nx[r], u[r]);
      Row8<GT>::unpack(ng[r], a[r]);
    }
    fetch(t0 + kTile);
    float A[VEC], H[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) A[i] = 1.f, H[i] = 0.f;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const bool in = t0 + wave * kSpan + group * kRows + r < s.len;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        float keep;
        const float d = decay_of<GATES>(a[r][i], lb[i], &keep);
        const float v = GATES ? keep * (u[r][i] * sigmoidf(u[r][i])) : u[r][i];
        a[r][i] = in ? d : 1.f;
        u[r][i] = in ? v : 0.f;
        H[i] = fmaf(a[r][i], H[i], u[r][i]);
        A[i] *= a[r][i];
      }
    }
    join_groups<true>(A, H, group);
    const float mine = join_waves<true>(sh, buf, A, H, group == kGroups - 1, wave, lane, &carry, &all);
    if (!OUT) continue;
    float h[VEC];
    spread(sh, mine, wave, lane, h);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float ea = __shfl_up(A[i], 8, 64), eh = __shfl_up(H[i], 8, 64);
      if (group > 0) h[i] = onto(ea, eh, h[i]);
    }
    if (p.states && group * kRows % kKept == 0) {
      const int64_t t = t0 + wave * kSpan + group * kRows;
      store8<float, WIDE>(p.states + (state_slot(s) + (s.c * p.segment + t) / kKept) * D + col, h, t < s.len ? valid : 0);
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int64_t t = t0 + wave * kSpan + group * kRows + r;
#pragma unroll
      for (int i = 0; i < VEC; ++i) h[i] = fmaf(a[r][i], h[i], u[r][i]);
      store8<T, WIDE>((T*)p.o + (s.begin + t) * D + col, h, t < s.len ? valid : 0);
    }
  }
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
template <typename T, typename GT, bool GATES, bool WIDE>
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
    lb[i] = GATES && p.lb && i < valid ? p.lb[col + i] : 0.f;
  }
  Row8<T>::unpack(rx, u);
  Row8<GT>::unpack(rg, a);
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    float keep;
    const float d = decay_of<GATES>(a[i], lb[i], &keep);
    h[i] = fmaf(d, h[i], GATES ? keep * (u[i] * sigmoidf(u[i])) : u[i]);
  }
  store8<T, WIDE>((T*)p.o + n * p.D + col, h, valid);
  if (p.ht) {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (i < valid) p.ht[n * p.D + col + i] = h[i];
  }
}

template <typename T, typename GT, bool GATES, bool WIDE>
int launch_fwd(const HgrnParams& p, int64_t segments, int64_t empty, hipStream_t st) {
  if (p.maps) {
    hipLaunchKernelGGL((hgrn_fwd_kernel<T, GT, GATES, WIDE, false>), dim3((unsigned)(segments * p.ncb)), dim3(kWaves * 64), 0, st, p);
    FLA_CHECK_LAUNCH();
  }
  hipLaunchKernelGGL((hgrn_fwd_kernel<T, GT, GATES, WIDE, true>), dim3((unsigned)((segments + empty) * p.ncb)), dim3(kWaves * 64), 0, st, p);
  FLA_CHECK_LAUNCH();
  return FLA_OK;
}

}  // namespace

extern "C" int64_t fla_hgrn_segment(int64_t n_seqs, int64_t tokens, int64_t longest, int64_t D) {
  if (n_seqs <= 0 || tokens <= 0 || longest <= 0 || D <= 0) return FLA_HGRN_TILE;
  const int64_t cbs = fla_cdiv(D, kCh), whole = fla_cdiv(longest, FLA_HGRN_TILE) * FLA_HGRN_TILE;
  // Whole sequences where they give every CU work of about the same length; otherwise four workgroups a CU, at most 64
  // segments to a sequence (a workgroup joins the maps of all segments ahead of its own).
  if (n_seqs * cbs >= 192 && longest * n_seqs <= 2 * tokens) return whole;
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
  const int64_t nseg = fla_cdiv(T, segment), cbs = fla_cdiv(D, kCh), segments = offsets ? NT : B * nseg;
  FLA_REQUIRE(maps || offsets || nseg == 1, FLA_E_INVALID);
  FLA_REQUIRE(D <= 0x3fffffff && (segments + N) <= 0x7fffffff / cbs, FLA_E_UNSUPPORTED);
  HgrnParams p{};
  p.x = x, p.g = g, p.lb = lower_bound, p.h0 = h0, p.o = o, p.ht = ht, p.states = states, p.maps = maps;
  p.offsets = offsets, p.indices = indices, p.chunk_offsets = chunk_offsets;
  p.NT = NT, p.segment = segment, p.T = T, p.ldx = ldx, p.ldg = ldg;
  p.D = (int)D, p.ncb = (int)cbs, p.nseg = (int)nseg;
  const bool wide = wide_rows(x, ldx, D, x_dtype) && wide_rows(g, ldg, D, g_dtype) && wide_rows(o, D, D, x_dtype);
  const int64_t empty = offsets ? N : 0;
  hipStream_t st = (hipStream_t)stream;
#define D_(XE, XT, GE, GT)                                                                                       \
  if (x_dtype == XE && g_dtype == GE) {                                                                          \
    if (gates) return wide ? launch_fwd<XT, GT, true, true>(p, segments, empty, st) : launch_fwd<XT, GT, true, false>(p, segments, empty, st); \
    return wide ? launch_fwd<XT, GT, false, true>(p, segments, empty, st) : launch_fwd<XT, GT, false, false>(p, segments, empty, st);         \
  }
  HGRN_TYPES(D_)
#undef D_
  return FLA_E_UNSUPPORTED;
}

extern "C" int fla_hgrn_step(const void* x, const void* g, const float* lower_bound, const float* h0, void* o, float* ht, int gates,
                             int x_dtype, int g_dtype, int64_t N, int64_t D, int64_t ldx, int64_t ldg, fla_stream_t stream) {
  FLA_REQUIRE(x && g && o && N > 0 && D > 0 && ldx >= D && ldg >= D && (!lower_bound || gates), FLA_E_INVALID);
  FLA_REQUIRE(D <= 0x3fffffff && N <= 0x7fffffff / fla_cdiv(D, VEC) , FLA_E_UNSUPPORTED);
  const StepParams p{x, g, lower_bound, h0, o, ht, N, ldx, ldg, (int)D};
  const bool wide = wide_rows(x, ldx, D, x_dtype) && wide_rows(g, ldg, D, g_dtype) && wide_rows(o, D, D, x_dtype);
  const dim3 grid((unsigned)fla_cdiv(N * fla_cdiv(D, VEC), 64));
  hipStream_t st = (hipStream_t)stream;
#define D_(XE, XT, GE, GT)                                                                                                   \
  if (x_dtype == XE && g_dtype == GE) {                                                                                      \
    if (gates && wide) hipLaunchKernelGGL((hgrn_step_kernel<XT, GT, true, true>), grid, dim3(64), 0, st, p);                 \
    else if (gates) hipLaunchKernelGGL((hgrn_step_kernel<XT, GT, true, false>), grid, dim3(64), 0, st, p);                   \
    else if (wide) hipLaunchKernelGGL((hgrn_step_kernel<XT, GT, false, true>), grid, dim3(64), 0, st, p);                    \
    else hipLaunchKernelGGL((hgrn_step_kernel<XT, GT, false, false>), grid, dim3(64), 0, st, p);                             \
    FLA_CHECK_LAUNCH();                                                                                                      \
    return FLA_OK;                                                                                                           \
  }
  HGRN_TYPES(D_)
#undef D_
  return FLA_E_UNSUPPORTED;
}
