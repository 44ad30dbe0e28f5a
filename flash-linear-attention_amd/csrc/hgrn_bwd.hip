// Backward of the elementwise gated recurrence.  With m_t the gradient that reaches h_t from later tokens, m_T = dht,
//   l_t = do_t + m_t,   m_{t-1} = a_t l_t,   dh0 = m_0,
//   log decays:       dx = l,            dg = l h_{t-1} a
//   pre-activations:  di = l (1-a) silu'(i),   da = l (h_{t-1} - silu(i)),   df = da (1-lb) s(1-s),   dlb = sum da (1-s)
// m runs from right to left through the scan of hgrn_scan.h with the maps m -> a (do + m).  h_{t-1} is formed again in fp32 from
// x, g and the states that the forward left ahead of every 16 rows (a wave's rows in a tile), so that it needs no scan across
// waves: the 16-bit o, which is what it would be read from otherwise, takes as many bytes and has lost half of the digits.
#include "hgrn_scan.h"

namespace {

// OUT: writes the gradients; otherwise the map of the segment.
template <typename T, typename GT, bool GATES, bool WIDE, bool OUT>
__global__ __launch_bounds__(kWaves * 64) void hgrn_bwd_kernel(HgrnParams p) {
  __shared__ __attribute__((aligned(16))) TileShare sh;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = lane >> 3;
  const int cb = blockIdx.x % p.ncb, D = p.D;
  bool exists;
  const Segment s = find_segment(p, blockIdx.x / p.ncb, &exists);
  if (!exists) return;
  const int ch = cb * kCh + lane;
  const int col = cb * kCh + (lane & 7) * VEC, valid = D - col;
  if (!OUT && s.c == 0) return;               // nothing is ahead of the first segment of a sequence
  float lb[VEC], dlb[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    lb[i] = GATES && p.lb && i < valid ? p.lb[col + i] : 0.f;
    dlb[i] = 0.f;
  }

  constexpr int kRows = kBwdRows, kSpan = kGroups * kRows, kTile = kWaves * kSpan;
  typename Row8<T>::raw nx[kRows], nd[kRows];
  typename Row8<GT>::raw ng[kRows];
  float nh[VEC];
  auto fetch = [&](int64_t t0) {
    const int64_t w0 = t0 + wave * kSpan;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int64_t t = w0 + group * kRows + r, row = s.begin + t;
      const int v = t >= 0 && t < s.len ? valid : 0;
      if (OUT) nx[r] = load_raw8<T, WIDE>((const T*)p.x + row * p.ldx + col, v);
      ng[r] = load_raw8<GT, WIDE>((const GT*)p.g + row * p.ldg + col, v);
      nd[r] = load_raw8<T, WIDE>((const T*)p.dout + row * D + col, p.dout ? v : 0);
    }
    if (OUT) {
      const bool v = t0 >= 0 && w0 < s.len;
      const float* st = p.states + (state_slot(s) + (s.c * p.segment + w0) / kKept) * D + col;
      Row8<float>::unpack(load_raw8<float, WIDE>(st, v ? valid : 0), nh);
    }
  };
  const int64_t last = s.len > 0 ? (s.len - 1) / kTile * kTile : -1;
  fetch(last);
  float carry = 0.f, all = 1.f;
  if (OUT && ch < D) {
    if (p.dht) carry = p.dht[s.n * D + ch];
    const float* m = p.maps + s.first * 2 * D + ch;
#pragma unroll 8
    for (int64_t k = s.count - 1; k > s.c; --k) carry = onto(m[2 * k * D], m[(2 * k + 1) * D], carry);
  }
  int buf = 0;
  for (int64_t t0 = last; t0 >= 0; t0 -= kTile, buf ^= 1) {
    float a[kRows][VEC], d[kRows][VEC], before[kRows][VEC], hs[VEC];
    typename Row8<T>::raw rx[kRows];
    typename Row8<GT>::raw rg[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      rx[r] = nx[r];
      rg[r] = ng[r];
      Row8<T>::unpack(nd[r], d[r]);
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) hs[i] = nh[i];
    fetch(t0 - kTile);

    float A[VEC], M[VEC];
    {
      // the lane's rows as a map of the state (H) and, from the right, of the gradient (M); before: u until the states are known
      float H[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) A[i] = 1.f, H[i] = 0.f, M[i] = 0.f;
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const bool in = t0 + wave * kSpan + group * kRows + r < s.len;
        float x[VEC], g[VEC];
        if (OUT) Row8<T>::unpack(rx[r], x);
        Row8<GT>::unpack(rg[r], g);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          float keep;
          const float dec = decay_of<GATES>(g[i], lb[i], &keep);
          a[r][i] = in ? dec : 1.f;
          if (OUT) {
            const float v = GATES ? keep * (x[i] * sigmoidf(x[i])) : x[i];
            before[r][i] = in ? v : 0.f;
            H[i] = fmaf(a[r][i], H[i], before[r][i]);
          }
          A[i] *= a[r][i];
        }
      }
#pragma unroll
      for (int r = kRows - 1; r >= 0; --r)
#pragma unroll
        for (int i = 0; i < VEC; ++i) M[i] = a[r][i] * (d[r][i] + M[i]);
      if (OUT) {
        float P[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) P[i] = A[i];
        join_groups<true>(P, H, group);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float ea = __shfl_up(P[i], 8, 64), eh = __shfl_up(H[i], 8, 64);
          float h = group > 0 ? onto(ea, eh, hs[i]) : hs[i];
#pragma unroll
          for (int r = 0; r < kRows; ++r) {
            const float u = before[r][i];
            before[r][i] = h;
            h = fmaf(a[r][i], h, u);
          }
        }
      }
    }
    join_groups<false>(A, M, group);
    const float mine = join_waves<false>(sh, buf, A, M, group == 0, wave, lane, &carry, &all);
    if (!OUT) continue;
    float m[VEC];
    spread(sh, mine, wave, lane, m);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float ea = __shfl_down(A[i], 8, 64), em = __shfl_down(M[i], 8, 64);
      if (group + 1 < kGroups) m[i] = onto(ea, em, m[i]);
    }
#pragma unroll
    for (int r = kRows - 1; r >= 0; --r) {
      const int64_t t = t0 + wave * kSpan + group * kRows + r, row = s.begin + t;
      const int v = t < s.len ? valid : 0;
      float x[VEC], g[VEC];
      if (GATES) {
        forget(rx[r]);
        forget(rg[r]);
      }
      Row8<T>::unpack(rx[r], x);
      Row8<GT>::unpack(rg[r], g);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float l = d[r][i] + m[i];
        m[i] = a[r][i] * l;
        if (GATES) {
          float sf, rest;
          sigmoid_both(g[i], &sf, &rest);
          const float si = sigmoidf(x[i]), z = x[i] * si;
          const float da = l * (before[r][i] - z);
          x[i] = l * (1.f - lb[i]) * rest * fmaf(z, 1.f - si, si);
          g[i] = da * (1.f - lb[i]) * sf * rest;
          dlb[i] += v > i ? da * rest : 0.f;
        } else {
          x[i] = l;
          g[i] = m[i] * before[r][i];
        }
      }
      store8<T, WIDE>((T*)p.dx + row * D + col, x, v);
      store8<GT, WIDE>((GT*)p.dg + row * D + col, g, v);
    }
  }
  if (wave == 0 && ch < D) {
    if (!OUT) {
      float* q = p.maps + s.id * 2 * D + ch;
      q[0] = all;
      q[D] = carry;
    } else if (p.dh0 && s.c == 0) {
      p.dh0[s.n * D + ch] = carry;
    }
  }
  if (OUT && p.dlb && s.len > 0) {   // the segment's column sums: the groups of a wave, then the waves in order
#pragma unroll
    for (int i = 0; i < VEC; ++i)
#pragma unroll
      for (int k = 8; k < 64; k *= 2) dlb[i] += __shfl_xor(dlb[i], k, 64);
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

template <typename T, typename GT, bool GATES, bool WIDE>
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
  const int64_t nseg = fla_cdiv(T, segment), cbs = fla_cdiv(D, kCh), segments = offsets ? NT : B * nseg;
  FLA_REQUIRE(maps || offsets || nseg == 1, FLA_E_INVALID);
  FLA_REQUIRE(D <= 0x3fffffff && (segments + N) <= 0x7fffffff / cbs, FLA_E_UNSUPPORTED);
  HgrnParams p{};
  p.x = x, p.g = g, p.lb = lower_bound, p.states = const_cast<float*>(states), p.maps = maps;
  p.dout = dout, p.dht = dht, p.dx = dx, p.dg = dg, p.dh0 = dh0, p.dlb = dlb_partials;
  p.offsets = offsets, p.indices = indices, p.chunk_offsets = chunk_offsets;
  p.NT = NT, p.segment = segment, p.T = T, p.ldx = ldx, p.ldg = ldg;
  p.D = (int)D, p.ncb = (int)cbs, p.nseg = (int)nseg;
  const bool wide = wide_rows(x, ldx, D, x_dtype) && wide_rows(g, ldg, D, g_dtype) && wide_rows(dout, D, D, x_dtype) &&
                    wide_rows(dx, D, D, x_dtype) && wide_rows(dg, D, D, g_dtype);
  const int64_t empty = offsets ? N : 0;
  hipStream_t st = (hipStream_t)stream;
#define D_(XE, XT, GE, GT)                                                                                       \
  if (x_dtype == XE && g_dtype == GE) {                                                                          \
    if (gates) return wide ? launch_bwd<XT, GT, true, true>(p, segments, empty, st) : launch_bwd<XT, GT, true, false>(p, segments, empty, st); \
    return wide ? launch_bwd<XT, GT, false, true>(p, segments, empty, st) : launch_bwd<XT, GT, false, false>(p, segments, empty, st);         \
  }
  HGRN_TYPES(D_)
#undef D_
  return FLA_E_UNSUPPORTED;
}
