// The router of route_groups.h by itself: four tokens to a workgroup, one to a wave.
#include "fp8.h"
#include "route_groups.h"

namespace vybdq {

template <bool SOFTMAX, bool BIAS, int TOP, int ENT>
__global__ void __launch_bounds__(256) k_route_groups(const RouteArgs a) {
  const int t = 4 * blockIdx.x + (threadIdx.x >> 6);
  if (t < a.T) route_groups_wave<SOFTMAX, BIAS, TOP, ENT>(a, t, nullptr);
}

int route_groups_args(const char *func, RouteArgs &a, uint64_t logits, int logits_dt, uint64_t bias, uint64_t idx, uint64_t w,
                      int64_t T, int64_t E, int64_t topk, double scale, int softmax, int renorm, int64_t groups,
                      int64_t top_groups, int64_t group_top) {
  auto bad = [&](int code, const char *msg) { return set_error(code, std::string(func) + ": " + msg); };
  if (!dt_valid_out(logits_dt)) return bad(VYBDQ_ERR_ARG, "logits_dt must be F32, F16, BF16 or F64");
  if (T < 0 || T >= (1 << 24) || E < 1 || E > 1024) return bad(VYBDQ_ERR_SHAPE, "need T below 2^24 and 1 <= E <= 1024");
  if (groups < 1 || groups > 64 || E % groups) return bad(VYBDQ_ERR_SHAPE, "groups must be in 1 .. 64 and divide E");
  if (top_groups < 1 || top_groups > groups) return bad(VYBDQ_ERR_SHAPE, "top_groups must be in 1 .. groups");
  if (group_top != 1 && group_top != 2) return bad(VYBDQ_ERR_ARG, "group_top must be 1 or 2");
  if (topk < 1 || topk > 64 || topk > top_groups * (E / groups))
    return bad(VYBDQ_ERR_SHAPE, "topk must be in 1 .. 64 and within the experts of top_groups groups");
  if (T > 0 && (!logits || !idx || !w)) return bad(VYBDQ_ERR_ARG, "null logits, idx_out or w_out");
  const int es = logits_dt == VYBDQ_F64 ? 8 : dt_size(logits_dt);
  if (logits % es || bias % 4 || idx % 4 || w % 4) return bad(VYBDQ_ERR_ALIGN, "buffers must be aligned to their elements");
  int lg = 6;
  while ((1 << (6 - lg)) < groups) --lg;
  a = RouteArgs{reinterpret_cast<const void *>(logits), logits_dt, reinterpret_cast<const float *>(bias), static_cast<int>(T),
                static_cast<int>(E), static_cast<int>(topk), static_cast<int>(groups), static_cast<int>(top_groups),
                static_cast<int>(group_top), softmax != 0, renorm != 0, static_cast<int>(E / groups), lg, scale,
                reinterpret_cast<int *>(idx), reinterpret_cast<float *>(w)};
  return VYBDQ_OK;
}

int route_groups_launch(const RouteArgs &a, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>((a.T + 3) / 4));
#define ROUTE(SM, BI, TP, ENT) hipLaunchKernelGGL((k_route_groups<SM, BI, TP, ENT>), grid, dim3(256), 0, s, a)
  VYBDQ_DISPATCH_ROUTE(a, ROUTE)
#undef ROUTE
  return check_launch("moe route (groups)");
}

}  // namespace vybdq

using namespace vybdq;

extern "C" int vybdq_moe_route_groups(uint64_t logits, int logits_dt, uint64_t bias, uint64_t idx_out, uint64_t w_out, int64_t T,
                                      int64_t E, int64_t topk, double scale, int softmax, int renorm, int64_t groups,
                                      int64_t top_groups, int64_t group_top, uint64_t stream) {
  RouteArgs a;
  const int rc = route_groups_args(__func__, a, logits, logits_dt, bias, idx_out, w_out, T, E, topk, scale, softmax, renorm,
                                   groups, top_groups, group_top);
  if (rc || T == 0) return rc;
  const Fp8Span in[2] = {fp8_bytes(logits, T * E * dt_size(logits_dt)), fp8_bytes(bias, 4 * E)};
  const Fp8Span i = fp8_bytes(idx_out, 4 * T * topk), w = fp8_bytes(w_out, 4 * T * topk);
  bool alias = fp8_overlap(i, w);
  for (const Fp8Span &r : in) alias = alias || fp8_overlap(r, i) || fp8_overlap(r, w);
  VYBDQ_REQUIRE(!alias, VYBDQ_ERR_ARG, "idx_out and w_out must not overlap each other, the logits or the bias");
  return route_groups_launch(a, as_stream(stream));
}
