// Backward of the elementwise gated recurrence.  With m_t the gradient that reaches h_t from later tokens, m_T = dht,
//   l_t = do_t + m_t,   m_{t-1} = a_t l_t,   dh0 = m_0,
//   log decays:       dx = l,            dg = l h_{t-1} a
//   pre-activations:  di = l (1-a) silu'(i),   da = l (h_{t-1} - silu(i)),   df = da (1-lb) s(1-s),   dlb = sum da (1-s)
// m runs from right to left through the scan of hgrn_scan.h with the maps m -> a (do + m).  h_{t-1} is formed again in fp32 from
// x, g and the states that the forward left ahead of every 16 rows (a wave's rows in a tile), so that it needs no scan across
// waves: the 16-bit o, which is what it would be read from otherwise, takes as many bytes and has lost half of the digits.
#include "hgrn_scan.h"

namespace {

// OUT: writes the gradients; otherwise the map of the segment.  A lane holds six values an element for the second half of a tile, 2 x 8 elements take
// all 256 registers: R = 4 does not fit.  On wide rows with gates the results' launch spills in eight instances (registers, bytes of scratch a
// lane): with a lower bound 14 (52) in 16 bits, 39 and 47 (136) with the gates in fp32, 119 (304) all in fp32; without one 1 (8) with the gates in
// fp32, 71 (192) all in fp32.  Its time on 8 x 4096 x 2048 (us; bf16, fp16, bf16 with fp32 gates, fp32; the bytes 133, 133, 185, 263): with a bound 190, 168, 212,
// 305; without 169, 162, 210, 278; log decays, which spill nowhere, 165, 156, 208, 280.  Joining both directions side by side, which hides one's shuffles
// behind the other's, spills more (227 instead of 188 with a bound in bf16; in 206 registers, with log decays, it takes as long as one after the other).
template <typename T, typename GT, int GATES, bool WIDE, bool OUT>
__global__ __launch_bounds__(kWaves * 64) void hgrn_bwd_kernel(HgrnParams p) {
  constexpr int R = 2, kSpan = kGroups * R, kTile = kWaves * kSpan;   // rows of a lane, a wave, the workgroup
  __shared__ __attribute__((aligned(16))) TileShare sh;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = lane >> 3;
  const int cb = blockIdx.x % p.ncb, D = p.D;
  bool exists;
  const Segment s = find_segment(p, blockIdx.x / p.ncb, &exists);
  if (!exists) return;
  if (!OUT && s.c == 0) return;               // nothing is ahead of the first segment of a sequence
  const int ch = cb * kCh + lane;
  const int col = cb * kCh + (lane & 7) * VEC, valid = D - col;
  if (GATES == kBoundedGates) keep_bounds(sh, p.lb, cb * kCh, D);
  float dlb[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) dlb[i] = 0.f;

  const int64_t row0 = s.begin + wave * kSpan;
  const T* xr = (const T*)p.x + row0 * p.ldx + cb * kCh;
  const GT* gr = (const GT*)p.g + row0 * p.ldg + cb * kCh;
  const int64_t out0 = row0 * D + cb * kCh;
  const uint32_t ax = lane_at<R>(lane, p.ldx), ag = lane_at<R>(lane, p.ldg), ao = lane_at<R>(lane, D);
  const float* st0 = p.states + (state_slot(s) + s.c * p.segment / kSpan + wave) * D + col;
  const int64_t left = s.len - wave * kSpan;
  typename Row8<T>::raw nx[R], nd[R];
  typename Row8<GT>::raw ng[R];
  typename Row8<float>::raw nh;
  auto fetch = [&](int64_t t0, auto full) {
    constexpr bool F = decltype(full)::value;
    const int64_t n = t0 < 0 ? 0 : left - t0;
    if (OUT) fetch_rows<T, WIDE, R, F>(nx, xr + t0 * p.ldx, p.ldx, ax, n, group, valid, 0.f);
    fetch_rows<GT, WIDE, R, F>(ng, gr + t0 * p.ldg, p.ldg, ag, n, group, valid, GATES ? __builtin_inff() : 0.f);
    fetch_rows<T, WIDE, R, F>(nd, (const T*)p.dout + out0 + t0 * D, D, ao, p.dout ? n : 0, group, valid, 0.f);
    if (OUT && F) nh = Row8<float>::load_raw(st0 + t0 / kKept * D);
    else if (OUT) nh = load_raw8<float, WIDE>(st0 + t0 / kKept * D, n > 0 ? valid : 0);
  };
  // tiles of which all rows and channels exist
  const int64_t whole = WIDE && cb * kCh + kCh <= D && p.dout ? s.len / kTile * kTile : 0;
  const int64_t last = s.len > 0 ? (s.len - 1) / kTile * kTile : -1;
  if (last >= 0 && last < whole) fetch(last, Full<true>());
  else fetch(last, Full<false>());
  float carry = 0.f, all = 1.f;
  if (OUT && ch < D) {
    if (p.dht) carry = p.dht[s.n * D + ch];
    const float* m = p.maps + s.first * 2 * D + ch;
#pragma unroll 4
    for (int64_t k = s.count - 1; k > s.c; --k) carry = onto(m[2 * k * D], m[(2 * k + 1) * D], carry);
  }
  int buf = 0;
  auto tile = [&](int64_t t0, auto full, auto full_next) {
    // Held for the second half: x itself, sigmoid(x), both sides of the forget gate's sigmoid (or the decay), do and the state ahead
    float x[R][VEC], si[R][VEC], sf[R][VEC], rest[R][VEC], d[R][VEC], before[R][VEC];
    float A[VEC], M[VEC], hs[VEC];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (OUT) Row8<T>::unpack(nx[r], x[r]);
      Row8<GT>::unpack(ng[r], sf[r]);
      Row8<T>::unpack(nd[r], d[r]);
    }
    if (OUT) Row8<float>::unpack(nh, hs);
    fetch(t0 - kTile, full_next);
    float lb[VEC];
    if (GATES == kBoundedGates) bounds_of(sh, lane, lb);
    auto decay = [&](int r, int i) { return GATES == kBoundedGates ? fmaf(1.f - lb[i], sf[r][i], lb[i]) : sf[r][i]; };
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        if (GATES) {
          sigmoid_both(sf[r][i], &sf[r][i], &rest[r][i]);
          if (OUT) si[r][i] = sigmoidf(x[r][i]);
        } else {
          sf[r][i] = __expf(sf[r][i]);
        }
      }
    auto weight = [&](int r, int i) { return GATES == kBoundedGates ? (1.f - lb[i]) * rest[r][i] : rest[r][i]; };   // 1 - a
    auto input = [&](int r, int i) { return GATES ? weight(r, i) * (x[r][i] * si[r][i]) : x[r][i]; };
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float a0 = decay(0, i), a1 = decay(1, i);
      A[i] = a0 * a1;
      M[i] = a0 * (d[0][i] + a1 * d[1][i]);
    }
    if (OUT) {
      float P[VEC], H[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        P[i] = A[i];
        H[i] = fmaf(decay(1, i), input(0, i), input(1, i));
      }
      join_groups<true>(P, H, group);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float ahead = __shfl_up(onto(P[i], H[i], hs[i]), 8, 64);
        before[0][i] = group > 0 ? ahead : hs[i];
        before[1][i] = fmaf(decay(0, i), before[0][i], input(0, i));
      }
    }
    join_groups<false>(A, M, group);
    const float mine = join_waves<false>(sh, buf, A, M, group == 0, wave, lane, &carry, &all);
    buf ^= 1;
    if (!OUT) return;
    const int64_t n = left - t0;
    if (!decltype(full)::value && n <= 0) return;   // (uniform, and no barrier behind it)
    float m[VEC];
    spread(sh, mine, wave, lane, m);
    if (GATES == kBoundedGates) bounds_of(sh, lane, lb);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float behind = __shfl_down(onto(A[i], M[i], m[i]), 8, 64);
      m[i] = group + 1 < kGroups ? behind : m[i];
    }
#pragma unroll
    for (int r = R - 1; r >= 0; --r) {
      float dx[VEC], dg[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float l = d[r][i] + m[i];
        m[i] = decay(r, i) * l;
        if (GATES) {
          const float z = x[r][i] * si[r][i], da = l * (before[r][i] - z);
          dx[i] = l * weight(r, i) * fmaf(z, 1.f - si[r][i], si[r][i]);
          dg[i] = da * weight(r, i) * sf[r][i];
          if (GATES == kBoundedGates) dlb[i] = fmaf(da, rest[r][i], dlb[i]);
        } else {
          dx[i] = l;
          dg[i] = m[i] * before[r][i];
        }
      }
      store_row<T, WIDE, R, decltype(full)::value>((T*)p.dx + out0 + t0 * D, D, ao, r, dx, n, group, valid);
      store_row<GT, WIDE, R, decltype(full)::value>((GT*)p.dg + out0 + t0 * D, D, ao, r, dg, n, group, valid);
    }
  };
  int64_t t0 = last;
  if (t0 >= whole && t0 >= 0) {   // the ragged end (or no tile is whole)
    if (whole > 0) tile(t0, Full<false>(), Full<true>()), t0 -= kTile;
    else
      for (; t0 >= 0; t0 -= kTile) tile(t0, Full<false>(), Full<false>());
  }
  for (; t0 > 0; t0 -= kTile) tile(t0, Full<true>(), Full<true>());
  if (t0 == 0) tile(t0, Full<true>(), Full<false>());
  if (wave == 0 && ch < D) {
    if (!OUT) {
      float* q = p.maps + s.id * 2 * D + ch;
      q[0] = all;
      q[D] = carry;
    } else if (p.dh0 && s.c == 0) {
      p.dh0[s.n * D + ch] = carry;
    }
  }
  if (OUT && GATES == kBoundedGates && p.dlb && s.len > 0) {   // the segment's column sums: the groups of a wave, then the waves in order
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
#pragma unroll
      for (int k = 8; k < 64; k *= 2) dlb[i] += __shfl_xor(dlb[i], k, 64);
    }
    __syncthreads();
    if (group == 0)
#pragma unroll
      for (int i = 0; i < VEC; ++i) sh.in[wave][lane * VEC + i] = dlb[i];
    __syncthreads();
    if (wave == 0 && ch < D) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) t += sh.in[w][lane];
      p.dlb[s.id * D + ch] = t;
    }
  }
}

template <typename T, typename GT, int GATES, bool WIDE>
int launch_bwd(const HgrnParams& p, int64_t segments, int64_t empty, hipStream_t st) {
  if (p.maps) {
    hipLaunchKernelGGL((hgrn_bwd_kernel<T, GT, GATES, WIDE, false>), dim3((unsigned)(segments * p.ncb)), dim3(kWaves * 64), 0, st, p);
    FLA_CHECK_LAUNCH();
  }
  hipLaunchKernelGGL((hgrn_bwd_kernel<T, GT, GATES, WIDE, true>), dim3((unsigned)((segments + empty) * p.ncb)), dim3(kWaves * 64), 0, st, p);
  FLA_CHECK_LAUNCH();
  return FLA_OK;
}

}  // namespace

extern "C" int fla_hgrn_bwd(const void* x, const void* g, const float* lower_bound, const float* states, const void* dout, const float* dht,
                            void* dx, void* dg, float* dh0, float* dlb_partials, float* maps, const int64_t* offsets,
                            const int64_t* indices, const int64_t* chunk_offsets, int64_t NT, int64_t segment, int gates, int x_dtype,
                            int g_dtype, int64_t B, int64_t T, int64_t D, int64_t N, int64_t ldx, int64_t ldg, fla_stream_t stream) {
  FLA_REQUIRE(x && g && states && dx && dg && B > 0 && T > 0 && D > 0 && N > 0 && NT >= 0 && ldx >= D && ldg >= D, FLA_E_INVALID);
  FLA_REQUIRE(segment > 0 && segment % FLA_HGRN_TILE == 0 && (!lower_bound || gates) && (!dlb_partials || lower_bound), FLA_E_INVALID);
  FLA_REQUIRE(offsets ? B == 1 && (indices || NT == 0) && chunk_offsets : N == B, FLA_E_INVALID);
  FLA_REQUIRE((uintptr_t)states % 16 == 0, FLA_E_ALIGNMENT);
  const int64_t nseg = fla_cdiv(T, segment), cbs = fla_cdiv(D, kCh), segments = offsets ? NT : B * nseg;
  FLA_REQUIRE(maps || offsets || nseg == 1, FLA_E_INVALID);
  FLA_REQUIRE(ldx <= FLA_HGRN_MAX_PITCH && ldg <= FLA_HGRN_MAX_PITCH && segments + N <= kMostWorkgroups / cbs, FLA_E_UNSUPPORTED);
  HgrnParams p{};
  p.x = x, p.g = g, p.lb = lower_bound, p.states = const_cast<float*>(states), p.maps = maps;
  p.dout = dout, p.dht = dht, p.dx = dx, p.dg = dg, p.dh0 = dh0, p.dlb = dlb_partials;
  p.offsets = offsets, p.indices = indices, p.chunk_offsets = chunk_offsets;
  p.NT = NT, p.segment = segment, p.T = T, p.ldx = ldx, p.ldg = ldg;
  p.D = (int)D, p.ncb = (int)cbs, p.nseg = (int)nseg;
  const bool wide = wide_rows(x, ldx, D, x_dtype) && wide_rows(g, ldg, D, g_dtype) && wide_rows(dout, D, D, x_dtype) &&
                    wide_rows(dx, D, D, x_dtype) && wide_rows(dg, D, D, g_dtype);
  const int64_t empty = offsets ? N : 0;
  const int kind = !gates ? kLogDecays : lower_bound ? kBoundedGates : kGates;
  hipStream_t st = (hipStream_t)stream;
#define D_(XE, XT, GE, GT)                                                                                       \
  if (x_dtype == XE && g_dtype == GE) {                                                                          \
    if (kind == kLogDecays) return wide ? launch_bwd<XT, GT, 0, true>(p, segments, empty, st) : launch_bwd<XT, GT, 0, false>(p, segments, empty, st); \
    if (kind == kGates) return wide ? launch_bwd<XT, GT, 1, true>(p, segments, empty, st) : launch_bwd<XT, GT, 1, false>(p, segments, empty, st); \
    return wide ? launch_bwd<XT, GT, 2, true>(p, segments, empty, st) : launch_bwd<XT, GT, 2, false>(p, segments, empty, st); \
  }
  HGRN_TYPES(D_)
#undef D_
  return FLA_E_UNSUPPORTED;
}
