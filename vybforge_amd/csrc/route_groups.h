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

__device__ __forceinline__ double shfl_xor_f64(double v, int d) { return __shfl_xor(v, d); }

// The larger of two doubles, NaN below every number.
__device__ __forceinline__ bool above(double a, double b) { return a > b || (a == a && b != b); }

template <int LDT, int ENT>
__device__ __forceinline__ void route_groups_wave(const RouteArgs &a, int t, int *__restrict__ idx_copy) {
  const int lane = threadIdx.x & 63, L = 1 << a.lg;
  const int g = lane >> a.lg, j = lane & (L - 1);
  const int64_t base = static_cast<int64_t>(t) * a.E;
  double l[ENT];
  uint32_t eid[ENT];
#pragma unroll
  for (int i = 0; i < ENT; ++i) {
    const int q = j + L * i;
    eid[i] = g < a.groups && q < a.S ? static_cast<uint32_t>(g * a.S + q) : kRouteNone;
    l[i] = eid[i] != kRouteNone ? load_logit<LDT>(a.logits, base + eid[i]) : 0.0;
  }
  double top = 0.0, sum = 0.0;  // softmax: the largest logit (0 where all are -infinity) and the sum of exp(l - top)
  if (a.softmax) {
    top = -INFINITY;
#pragma unroll
    for (int i = 0; i < ENT; ++i)
      if (eid[i] != kRouteNone) top = l[i] > top || l[i] != l[i] ? l[i] : top;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const double o = shfl_xor_f64(top, d);
      top = o > top || o != o ? o : top;
    }
    if (top == -INFINITY) top = 0.0;
#pragma unroll
    for (int i = 0; i < ENT; ++i)
      if (eid[i] != kRouteNone) sum += exp(l[i] - top);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum += shfl_xor_f64(sum, d);
  }
  auto score = [&](double x) {
    if (!a.softmax) return 1.0 / (1.0 + exp(-x));
    return sum == 0.0 ? 0.0 : exp(x - top) / sum;
  };
  const bool sums = a.groups > 1 && a.group_top == 2;  // group values need the scores themselves
  uint64_t key[ENT];
  double b1 = -INFINITY, b2 = -INFINITY;  // this lane's best two choices (of how many: n)
  int n = 0;
#pragma unroll
  for (int i = 0; i < ENT; ++i) {
    key[i] = 0;
    if (eid[i] == kRouteNone) continue;
    double c = l[i];
    if (a.bias) c = score(c) + static_cast<double>(a.bias[eid[i]]);
    key[i] = double_order_key(c);
    if (a.groups > 1) {
      if (sums && !a.bias) c = score(c);
      if (n == 0 || above(c, b1)) {
        b2 = n ? b1 : b2;
        b1 = c;
      } else if (n == 1 || above(c, b2)) {
        b2 = c;
      }
      ++n;
    }
  }
  if (a.groups > 1) {
    for (int d = 1; d < L; d <<= 1) {
      const double o1 = shfl_xor_f64(b1, d), o2 = shfl_xor_f64(b2, d);
      const int on = __shfl_xor(n, d);
      // merge two descending pairs of which the first n and on entries (at most two) count
      const bool mine = n > 0 && (on == 0 || !above(o1, b1));
      const double f = mine ? b1 : o1;
      const double x = mine ? b2 : b1, y = mine ? o1 : o2;  // candidates for the second place
      const bool hx = mine ? n > 1 : n > 0, hy = mine ? on > 0 : on > 1;
      b2 = hx && (!hy || !above(y, x)) ? x : y;
      b1 = f;
      n = n + on;
    }
    double value = b1;
    if (a.group_top == 2 && n > 1) value = b1 + b2;
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
  const uint32_t mine = route_select<ENT>(key, eid, a.topk);
  const bool slot = lane < a.topk && mine != kRouteNone;
  const double sc = slot ? score(load_logit<LDT>(a.logits, base + mine)) : 0.0;
  double den = 1.0;
  if (a.renorm) {
    const uint64_t sb = __double_as_longlong(sc);
    double tot = 0.0;  // in slot order
    for (int q = 0; q < a.topk; ++q) {
      const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(sb), q);
      const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(sb >> 32), q);
      tot += __longlong_as_double(static_cast<long long>((static_cast<uint64_t>(hi) << 32) | lo));
    }
    den = tot + 1e-20;
  }
  if (slot) {
    const int64_t at = static_cast<int64_t>(t) * a.topk + lane;
    a.idx[at] = static_cast<int>(mine);
    a.w[at] = static_cast<float>(sc / den * a.scale);
    if (idx_copy) idx_copy[at] = static_cast<int>(mine);
  }
}

// experts per lane: 4, 8, 16 or 32
inline int route_groups_ent(const RouteArgs &a) {
  const int n = (a.S + (1 << a.lg) - 1) >> a.lg;
  return n <= 4 ? 4 : n <= 8 ? 8 : n <= 16 ? 16 : 32;
}

#define VYBDQ_DISPATCH_ROUTE(a, ...)                                              \
  switch (route_groups_ent(a)) {                                                 \
    case 4: { constexpr int ENT = 4; __VA_ARGS__; } break;                       \
    case 8: { constexpr int ENT = 8; __VA_ARGS__; } break;                       \
    case 16: { constexpr int ENT = 16; __VA_ARGS__; } break;                     \
    default: { constexpr int ENT = 32; __VA_ARGS__; } break;                     \
  }

// Checks the arguments and fills `a`; `func` names the entry point in errors.
int route_groups_args(const char *func, RouteArgs &a, uint64_t logits, int logits_dt, uint64_t bias, uint64_t idx, uint64_t w,
                      int64_t T, int64_t E, int64_t topk, double scale, int softmax, int renorm, int64_t groups,
                      int64_t top_groups, int64_t group_top);
int route_groups_launch(const RouteArgs &a, hipStream_t s);

}  // namespace vybdq
