// vybdq_kv_attn: checks, the choice of variant and key split, and the dispatch (kernel: kv_attn.h).
#include "kv_attn.h"

#include <string>

namespace vybdq {

// kv_attn_h.hip (fp16 / bf16 queries), kv_attn_f.hip (float32 queries, two fp16 terms)
void kv_attn_launch_h(int D, int variant, const KvAttnArgs &a, dim3 grid, hipStream_t s);
void kv_attn_launch_f(int D, int variant, const KvAttnArgs &a, dim3 grid, hipStream_t s);

constexpr int64_t kKvPartRows = 65536;   // rows of split results that a workspace holds
constexpr int64_t kKvArrivalBytes = 16384;

}  // namespace vybdq

using namespace vybdq;

extern "C" int64_t vybdq_kv_attn_workspace_size(int64_t D) {
  if (!(D == 64 || D == 128 || D == 192 || D == 256)) return -1;
  return kKvArrivalBytes + kKvPartRows * (D + 2) * 4;
}

extern "C" int vybdq_kv_attn(uint64_t K, uint64_t V, uint64_t Ks, uint64_t Vs, int64_t n_pages, int64_t Hkv, int64_t D,
                             int64_t page, uint64_t q, int x_dt, int64_t ldq, int64_t Hq, uint64_t out, uint64_t lse,
                             uint64_t table, int64_t W, uint64_t q_start, uint64_t ctx, int64_t T, int64_t B,
                             int64_t max_new, int64_t max_ctx, double scale, int causal, int64_t window, uint64_t ws,
                             int64_t ws_bytes, uint64_t stream) {
  VYBDQ_REQUIRE(dt_valid_in(x_dt), VYBDQ_ERR_ARG, "x_dt must be F32, F16 or BF16");
  VYBDQ_REQUIRE(D == 64 || D == 128 || D == 192 || D == 256, VYBDQ_ERR_SHAPE, "D must be 64, 128, 192 or 256");
  VYBDQ_REQUIRE(page >= 16 && page <= 256 && (page & (page - 1)) == 0, VYBDQ_ERR_SHAPE,
                "page must be a power of two in 16 .. 256");
  VYBDQ_REQUIRE(n_pages >= 1 && n_pages < (int64_t(1) << 31), VYBDQ_ERR_SHAPE, "n_pages must be in 1 .. 2^31 - 1");
  VYBDQ_REQUIRE(Hkv >= 1 && Hkv <= 1024 && Hq >= Hkv && Hq % Hkv == 0 && Hq <= 16384, VYBDQ_ERR_SHAPE,
                "Hq must be a multiple of Hkv, Hkv in 1 .. 1024 and Hq at most 16384");
  VYBDQ_REQUIRE(T >= 0 && T < (int64_t(1) << 30) && B >= 0 && B < (int64_t(1) << 20), VYBDQ_ERR_SHAPE,
                "T must be below 2^30 and B below 2^20");
  VYBDQ_REQUIRE(W >= 1 && W * page < (int64_t(1) << 30), VYBDQ_ERR_SHAPE, "W must be at least 1 and W * page below 2^30");
  VYBDQ_REQUIRE(window >= 0 && window < (int64_t(1) << 30), VYBDQ_ERR_SHAPE, "window must be in 0 .. 2^30 - 1");
  if (T == 0 || B == 0) return VYBDQ_OK;
  VYBDQ_REQUIRE(K && V && Ks && Vs && q && out && table && q_start && ctx, VYBDQ_ERR_ARG, "null pointer");
  VYBDQ_REQUIRE(ldq >= Hq * D, VYBDQ_ERR_SHAPE, "a row stride is smaller than a row");
  VYBDQ_REQUIRE((K | V | q | out) % 16 == 0 && ldq * dt_size(x_dt) % 16 == 0, VYBDQ_ERR_ALIGN,
                "codes, rows and out must be 16-byte aligned");
  VYBDQ_REQUIRE((Ks | Vs | table | q_start | ctx | lse) % 4 == 0, VYBDQ_ERR_ALIGN,
                "scales, table, q_start, ctx and lse must be 4-byte aligned");
  VYBDQ_REQUIRE(!ws || ws % 256 == 0, VYBDQ_ERR_ALIGN, "the workspace must be 256-byte aligned");
  int ps = 4;
  while ((1 << ps) < page) ++ps;
  const int G = static_cast<int>(Hq / Hkv);
  const bool two = x_dt == VYBDQ_F32;
  // Variant: 0, 1: 16 or 32 query rows, the waves of a workgroup take turns over the keys; 2: rows spread over
  // the waves (kv_attn_*.hip).
  const int64_t rows = max_new >= 1 ? max_new * G : T * G;
  const int variant = rows <= 16 ? 0 : rows <= 32 ? 1 : 2;
  const int64_t R = variant == 0 ? 16 : variant == 1 ? 32 : two && D > 128 ? 64 : 128;
  KvAttnArgs a{};
  a.per_seq = variant < 2;
  const int64_t units = a.per_seq ? B : T * G / R + B;
  VYBDQ_REQUIRE(units * Hkv < (int64_t(1) << 31), VYBDQ_ERR_SHAPE, "too many rows in one call");
  // Keys split over workgroups until the chip is full: at least 8 steps of 32 keys each, and what the workspace holds
  const int64_t wgs = units * Hkv, cap = W * page;
  const int64_t tokens = max_ctx >= 1 && max_ctx < cap ? max_ctx : cap;
  const int64_t steps = (tokens + 31) / 32;
  int64_t S = 1;
  if (ws && ws_bytes > kKvArrivalBytes && wgs * 4 <= kKvArrivalBytes) {
    const int64_t held = (ws_bytes - kKvArrivalBytes) / (R * (D + 2) * 4);
    const int64_t want = 4 * static_cast<int64_t>(device_cu_count()) / (variant == 2 ? 2 : 1);
    S = want / wgs;
    if (S > steps / 8) S = steps / 8;
    if (S > held / wgs) S = held / wgs;
    if (S < 1) S = 1;
  }
  const int rc = kv_status_address(a.b.status);
  if (rc) return rc;
  uint32_t *status = a.b.status;
  a.c = {reinterpret_cast<uint8_t *>(K), reinterpret_cast<uint8_t *>(V), reinterpret_cast<float *>(Ks),
         reinterpret_cast<float *>(Vs), static_cast<int32_t>(n_pages), static_cast<int32_t>(Hkv), ps};
  a.b = {reinterpret_cast<const int32_t *>(table), reinterpret_cast<const int32_t *>(q_start),
         reinterpret_cast<const int32_t *>(ctx), status, W, static_cast<int32_t>(T), static_cast<int32_t>(B)};
  a.q = reinterpret_cast<const void *>(q);
  a.out = reinterpret_cast<void *>(out);
  a.lse = reinterpret_cast<float *>(lse);
  a.arrivals = reinterpret_cast<uint32_t *>(ws);
  a.part = reinterpret_cast<float *>(ws + kKvArrivalBytes);
  a.ldq = ldq;
  a.G = G;
  a.dt = x_dt;
  a.causal = causal != 0;
  a.window = static_cast<int32_t>(window);
  a.scale2 = static_cast<float>(scale * 1.4426950408889634);
  const dim3 grid(static_cast<unsigned>(wgs), static_cast<unsigned>(S));
  if (two) kv_attn_launch_f(static_cast<int>(D), variant, a, grid, as_stream(stream));
  else kv_attn_launch_h(static_cast<int>(D), variant, a, grid, as_stream(stream));
  return check_launch("vybdq_kv_attn");
}
