// The router with softmax or sigmoid scores, experts in groups and a choice of groups, gfx950.
//
//   score = sigmoid(l) or softmax(l) over all E;  choice = score + bias
//   group g holds experts g S .. g S + S - 1 (S = E / groups); its value is the sum of its group_top (1 or 2) best choices;
//   the top_groups best groups stay; idx = the topk best choices in them; w = score[idx] (/ (sum + 1e-20)) * scale
//   every order is descending with ties to the lower id; scores, choices and values are float64.
// Without a bias a choice is compared by its logit (both scores rise with it: the exact order, where scores saturate too).
// NaN choices and values come below every number. A softmax over nothing but -infinity has scores 0.
//
// One wave takes a token. Lane j of the L = 64 / (groups rounded up to a power of two) lanes of group g holds its experts
// g S + j + L i, i < ENT, so a group's best two are a lane's best two, then log2 L steps over lanes.
#pragma once
#include "moe_route.h"

namespace vybdq {

struct RouteArgs {
  const void *logits;
  int ldt;
  const float *bias;
  int T, E, topk, groups, top_groups, group_top, softmax, renorm;
  int S, lg;  // experts to a group, log2 of the lanes to a group
  double scale;
  int *idx;
  float *w;
};

// exp(x) in float64, about an ulp off: x = n ln 2 + r with |r| <= ln 2 / 2 (Cody and Waite: ln 2 in two parts, so that r is
// exact to float64), the Taylor series of r to r^13 (the rest is below 2^-57), times 2^n. No special cases but the clamp: a NaN
// passes, below -745 the result is 0, above 710 infinity. (The library's exp and its tests of the range, at every place that
// a template argument does not decide, made the router 2500 instructions; it is 800 to a token of 160 experts so.)
__device__ __forceinline__ double route_exp(double x) {
  x = x < -800.0 ? -800.0 : (x > 800.0 ? 800.0 : x);
  const double n = __builtin_rint(x * 1.4426950408889634);
  double r = fma(n, -0x1.62e42feep-1, x);          // the leading 32 bits of ln 2: n of them are exact
  r = fma(n, -0x1.a39ef35793c76p-33, r);           // the rest of it
  double p = 1.0 / 6227020800.0;
  p = fma(p, r, 1.0 / 479001600.0);
  p = fma(p, r, 1.0 / 39916800.0);
  p = fma(p, r, 1.0 / 3628800.0);
  p = fma(p, r, 1.0 / 362880.0);
  p = fma(p, r, 1.0 / 40320.0);
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return __builtin_ldexp(p, static_cast<int>(n));
}

// The value of the lane that DPP control C names (every lane has one), and of lane l.
template <int C>
__device__ __forceinline__ double dpp_f64(double v) {
  const uint64_t b = __double_as_longlong(v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(b), C, 0xf, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(b >> 32), C, 0xf, 0xf, false);
  return __longlong_as_double(static_cast<long long>((static_cast<uint64_t>(hi) << 32) | lo));
}
__device__ __forceinline__ double lane_f64(double v, int l) {
  const uint64_t b = __double_as_longlong(v);
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(b), l), hi = __builtin_amdgcn_readlane(static_cast<int>(b >> 32), l);
  return __longlong_as_double(static_cast<long long>((static_cast<uint64_t>(hi) << 32) | lo));
}

// op over the wave: the rows of 16 by DPP, then the four rows.
template <class F>
__device__ __forceinline__ double wave_f64(double v, F op) {
  v = op(v, dpp_f64<DPP_QUAD_XOR1>(v));
  v = op(v, dpp_f64<DPP_QUAD_XOR2>(v));
  v = op(v, dpp_f64<DPP_HALF_MIRROR>(v));
  v = op(v, dpp_f64<DPP_ROW_MIRROR>(v));
  return op(op(lane_f64(v, 0), lane_f64(v, 16)), op(lane_f64(v, 32), lane_f64(v, 48)));
}

// The same selection as route_select, for up to 8 entries a lane: each lane sorts its entries once (best first, ties to the lower
// id; Batcher's odd-even merge), so a round compares the lanes' first entries and the winner's lane moves up (16384 tokens over 160
// experts in groups, 6 to a token: 25.6 us with the entries compared anew each round, 22.3 to 23.7 so).
template <int ENT>
__device__ __forceinline__ uint32_t route_select_sorted(uint64_t (&key)[ENT], uint32_t (&eid)[ENT], int topk) {
  static_assert(ENT == 4 || ENT == 8, "sorting networks");
  constexpr int kSwaps = ENT == 4 ? 5 : 19;
  constexpr int kA[2][19] = {{0, 2, 0, 1, 1}, {0, 2, 4, 6, 0, 1, 4, 5, 1, 5, 0, 1, 2, 3, 2, 3, 1, 3, 5}};
  constexpr int kB[2][19] = {{1, 3, 2, 3, 2}, {1, 3, 5, 7, 2, 3, 6, 7, 2, 6, 4, 5, 6, 7, 4, 5, 2, 4, 6}};
#pragma unroll
  for (int c = 0; c < kSwaps; ++c) {
    const int x = kA[ENT == 8][c], y = kB[ENT == 8][c];
    const bool swap = (key[y] > key[x]) | ((key[y] == key[x]) & (eid[y] < eid[x]));
    const uint64_t k = key[x];
    const uint32_t e = eid[x];
    key[x] = swap ? key[y] : k;
    key[y] = swap ? k : key[y];
    eid[x] = swap ? eid[y] : e;
    eid[y] = swap ? e : eid[y];
  }
  const int lane = threadIdx.x & 63;
  uint32_t mine = kRouteNone;  // lane s < topk: the expert of slot s
  for (int s = 0; s < topk; ++s) {
    const uint32_t khi = static_cast<uint32_t>(key[0] >> 32), mhi = wave_ext_u32<true>(khi);
    uint64_t own = __ballot(khi == mhi && eid[0] != kRouteNone);
    if (__popcll(own) > 1) {
      const uint32_t klo = khi == mhi ? static_cast<uint32_t>(key[0]) : 0u;
      const uint32_t mlo = wave_ext_u32<true>(klo);
      const uint32_t e1 = wave_ext_u32<false>(khi == mhi && klo == mlo ? eid[0] : kRouteNone);
      own = __ballot(eid[0] == e1 && e1 != kRouteNone);
    }
    const int src = own ? static_cast<int>(__builtin_ctzll(own)) : 0;
    const uint32_t we = own ? static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(eid[0]), src)) : kRouteNone;
    mine = lane == s ? we : mine;
    const bool won = lane == src;
#pragma unroll
    for (int i = 0; i < ENT; ++i) {
      key[i] = won ? (i + 1 < ENT ? key[i + 1 < ENT ? i + 1 : i] : 0) : key[i];
      eid[i] = won ? (i + 1 < ENT ? eid[i + 1 < ENT ? i + 1 : i] : kRouteNone) : eid[i];
    }
  }
  return mine;
}

// TOP: 0 without groups, else the choices that a group's value sums. A NaN stands for no entry and lies below every number (as
// fmax has it).
template <bool SOFTMAX, bool BIAS, int TOP, int ENT>
__device__ __forceinline__ void route_groups_wave(const RouteArgs &a, int t, int *__restrict__ idx_copy) {
  constexpr bool SCORES = SOFTMAX || BIAS || TOP == 2;  // every expert's score is needed, not the winners' alone
  constexpr bool LATE = SOFTMAX && !BIAS && TOP < 2;    // softmax: only the winners' are divided by the sum
  const int lane = threadIdx.x & 63, L = TOP ? 1 << a.lg : 64;
  const int g = TOP ? lane >> a.lg : 0, j = lane & (L - 1), S = TOP ? a.S : a.E;
  const int64_t base = static_cast<int64_t>(t) * a.E;
  auto logit = [&](int64_t i) {
    switch (a.ldt) {
      case VYBDQ_F64: return load_logit<VYBDQ_F64>(a.logits, i);
      case VYBDQ_F32: return load_logit<VYBDQ_F32>(a.logits, i);
      case VYBDQ_F16: return load_logit<VYBDQ_F16>(a.logits, i);
      default: return load_logit<VYBDQ_BF16>(a.logits, i);
    }
  };
  const double kNan = __longlong_as_double(0x7ff8000000000000ll);
  double l[ENT], bias[ENT], score[ENT], sum = 1.0;
  uint32_t eid[ENT];
#pragma unroll
  for (int i = 0; i < ENT; ++i) {
    const int q = j + L * i;
    const bool have = (TOP == 0 || g < a.groups) && q < S;
    eid[i] = have ? static_cast<uint32_t>(g * S + q) : kRouteNone;
    const uint32_t at = have ? eid[i] : 0;
    l[i] = logit(base + at);
    bias[i] = BIAS ? static_cast<double>(a.bias[at]) : 0.0;
    score[i] = 0.0;
  }
  if constexpr (SOFTMAX) {
    // the largest logit (0 where all are -infinity; NaN if one is), exp(l - top) over their sum
    double top = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < ENT; ++i) {
      top = eid[i] != kRouteNone ? fmax(top, l[i]) : top;
      nan |= eid[i] != kRouteNone && l[i] != l[i];
    }
    top = wave_f64(top, [](double x, double y) { return fmax(x, y); });
    if (top == -INFINITY) top = 0.0;
    if (__any(nan)) top = kNan;
    sum = 0.0;
#pragma unroll
    for (int i = 0; i < ENT; ++i) {
      score[i] = eid[i] != kRouteNone ? route_exp(l[i] - top) : 0.0;
      sum += score[i];
    }
    sum = wave_f64(sum, [](double x, double y) { return x + y; });
#pragma unroll
    for (int i = 0; i < ENT && !LATE; ++i) score[i] = sum == 0.0 ? 0.0 : score[i] / sum;
  } else if constexpr (SCORES) {
#pragma unroll
    for (int i = 0; i < ENT; ++i) score[i] = 1.0 / (1.0 + route_exp(-l[i]));
  }
  uint64_t key[ENT];
  double b1 = kNan, b2 = kNan;  // this lane's best two choices
#pragma unroll
  for (int i = 0; i < ENT; ++i) {
    const bool have = eid[i] != kRouteNone;
    const double order = BIAS ? score[i] + bias[i] : l[i];
    key[i] = have ? double_order_key(order) : 0;
    if constexpr (TOP > 0) {
      const double c = have ? (TOP == 2 && !BIAS ? score[i] : order) : kNan;
      if (TOP == 2) b2 = fmax(b2, b1 == b1 && c == c ? fmin(b1, c) : kNan);
      b1 = fmax(b1, c);
    }
  }
  if constexpr (TOP > 0) {
    auto merge = [&](double o1, double o2) {
      if (TOP == 2) b2 = fmax(b1 == b1 && o1 == o1 ? fmin(b1, o1) : kNan, fmax(b2, o2));
      b1 = fmax(b1, o1);
    };
    // (the lanes of a quad, then of a half row agree by then: a mirror's lane holds what lane ^ 4, ^ 8 does)
    if (a.lg > 0) merge(dpp_f64<DPP_QUAD_XOR1>(b1), TOP == 2 ? dpp_f64<DPP_QUAD_XOR1>(b2) : 0.0);
    if (a.lg > 1) merge(dpp_f64<DPP_QUAD_XOR2>(b1), TOP == 2 ? dpp_f64<DPP_QUAD_XOR2>(b2) : 0.0);
    if (a.lg > 2) merge(dpp_f64<DPP_HALF_MIRROR>(b1), TOP == 2 ? dpp_f64<DPP_HALF_MIRROR>(b2) : 0.0);
    if (a.lg > 3) merge(dpp_f64<DPP_ROW_MIRROR>(b1), TOP == 2 ? dpp_f64<DPP_ROW_MIRROR>(b2) : 0.0);
    if (a.lg > 4) merge(__shfl_xor(b1, 16), TOP == 2 ? __shfl_xor(b2, 16) : 0.0);
    const double value = TOP == 2 && S > 1 ? b1 + b2 : b1;
    uint64_t gk[1] = {0};
    uint32_t gi[1] = {kRouteNone};
    if (j == 0 && g < a.groups) {
      gk[0] = double_order_key(value);
      gi[0] = static_cast<uint32_t>(g);
    }
    const uint32_t kept = route_select<1>(gk, gi, a.top_groups);
    bool in = false;
    for (int s = 0; s < a.top_groups; ++s)
      in |= static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(kept), s)) == static_cast<uint32_t>(g);
#pragma unroll
    for (int i = 0; i < ENT; ++i) {
      eid[i] = in ? eid[i] : kRouteNone;
      key[i] = in ? key[i] : 0;
    }
  }
  uint32_t mine;
  if constexpr (ENT <= 8) mine = route_select_sorted<ENT>(key, eid, a.topk);
  else mine = route_select<ENT>(key, eid, a.topk);
  const bool slot = lane < a.topk && mine != kRouteNone;
  double sc = 0.0;
  if constexpr (SCORES && ENT <= 8) {  // from the lane and entry that hold the expert
    const int e = slot ? static_cast<int>(mine) : 0, gq = TOP ? e / S : 0, q = e - gq * S;
    const int from = TOP ? (gq << a.lg) + (q & (L - 1)) : q & 63, at = TOP ? q >> a.lg : q >> 6;
#pragma unroll
    for (int i = 0; i < ENT; ++i) {
      const double v = __shfl(score[i], from);
      sc = at == i ? v : sc;
    }
    sc = slot ? sc : 0.0;
  } else if constexpr (SOFTMAX) {
    for (int s = 0; s < a.topk; ++s) {  // the lane that holds slot s's expert gives its score
      const uint32_t e = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(mine), s));
      const int gq = TOP ? static_cast<int>(e) / S : 0, q = static_cast<int>(e) - gq * S;
      const int from = TOP ? (gq << a.lg) + (q & (L - 1)) : q & 63, at = TOP ? q >> a.lg : q >> 6;
      double v = 0.0;
#pragma unroll
      for (int i = 0; i < ENT; ++i) v = at == i ? score[i] : v;
      v = lane_f64(v, from & 63);
      sc = lane == s ? v : sc;
    }
  } else {
    sc = slot ? 1.0 / (1.0 + route_exp(-logit(base + mine))) : 0.0;
  }
  if constexpr (LATE) sc = sum == 0.0 ? 0.0 : sc / sum;
  double den = 1.0;
  if (a.renorm) {
    double tot = 0.0;  // in slot order
    for (int q = 0; q < a.topk; ++q) tot += lane_f64(sc, q);
    den = tot + 1e-20;
  }
  if (slot) {
    const int64_t at = static_cast<int64_t>(t) * a.topk + lane;
    a.idx[at] = static_cast<int>(mine);
    a.w[at] = static_cast<float>(sc / den * a.scale);
    if (idx_copy) idx_copy[at] = static_cast<int>(mine);
  }
}

// experts per lane: 4, 8 or 32
inline int route_groups_ent(const RouteArgs &a) {
  const int n = (a.S + (1 << a.lg) - 1) >> a.lg;
  return n <= 4 ? 4 : n <= 8 ? 8 : 32;
}

// Runs BODY(SOFTMAX, BIAS, TOP, ENT) with the arguments' template values.
#define VYBDQ_ROUTE_ENT(a, BODY, SM, BI, TP)                  \
  switch (route_groups_ent(a)) {                             \
    case 4: BODY(SM, BI, TP, 4); break;                      \
    case 8: BODY(SM, BI, TP, 8); break;                      \
    default: BODY(SM, BI, TP, 32); break;                    \
  }
#define VYBDQ_ROUTE_TOP(a, BODY, SM, BI)                      \
  switch ((a).groups == 1 ? 0 : (a).group_top) {             \
    case 0: VYBDQ_ROUTE_ENT(a, BODY, SM, BI, 0) break;       \
    case 1: VYBDQ_ROUTE_ENT(a, BODY, SM, BI, 1) break;       \
    default: VYBDQ_ROUTE_ENT(a, BODY, SM, BI, 2) break;      \
  }
#define VYBDQ_DISPATCH_ROUTE(a, BODY)                         \
  switch (((a).softmax ? 2 : 0) + ((a).bias ? 1 : 0)) {      \
    case 0: VYBDQ_ROUTE_TOP(a, BODY, false, false) break;    \
    case 1: VYBDQ_ROUTE_TOP(a, BODY, false, true) break;     \
    case 2: VYBDQ_ROUTE_TOP(a, BODY, true, false) break;     \
    default: VYBDQ_ROUTE_TOP(a, BODY, true, true) break;     \
  }

// Checks the arguments and fills `a`; `func` names the entry point in errors.
int route_groups_args(const char *func, RouteArgs &a, uint64_t logits, int logits_dt, uint64_t bias, uint64_t idx, uint64_t w,
                      int64_t T, int64_t E, int64_t topk, double scale, int softmax, int renorm, int64_t groups,
                      int64_t top_groups, int64_t group_top);
int route_groups_launch(const RouteArgs &a, hipStream_t s);

}  // namespace vybdq
