// vybdq_kv_attn: checks, the choice of variant and key split, and the dispatch (kernel: kv_attn.h).
#include "kv_attn.h"

#include <cmath>
#include <cstdlib>
#include <string>

namespace vybdq {

// kv_attn_h.hip (fp16 / bf16 queries), kv_attn_f.hip (float32 queries, two fp16 terms)
void kv_attn_launch_h(int D, int variant, const KvAttnArgs &a, dim3 grid, hipStream_t s);
void kv_attn_launch_f(int D, int variant, const KvAttnArgs &a, dim3 grid, hipStream_t s);

constexpr int64_t kKvPartRows = 131072;  // rows of split results that a workspace holds
constexpr int64_t kKvArrivalBytes = 16384;
// Keys to a split at most. A lane adds a split's weights four at a time, a matrix instruction's sum those of 32: 2^20 and 2^19
// float32 additions here. Of equal weights each is rounded alike, by up to 2^-24 of the sum so far: 2^-5 of one of them at the
// end. (From 2^24 additions on nothing is added any more: 2^29 keys in one split gave half their sum.)
constexpr int64_t kKvSplitKeys = int64_t(1) << 24;

struct KvShape {
  int64_t D, Hkv, G, T, B, new_rows, tokens;  // new_rows, tokens: most rows and most keys of a sequence
  bool two, causal;
  int64_t window, part_rows;  // part_rows: rows of split results that the workspace holds
};
struct KvPlan {
  int variant;
  int64_t units, splits;
  double time;
  bool by_length;  // k_kv_attn_keys: more splits for longer sequences
};

// The most keys that a tile of R rows reads.
static int64_t kv_keys(const KvShape &s, int64_t R) {
  return s.window && s.window + R / s.G < s.tokens ? s.window + R / s.G : s.tokens;
}

// How many splits fit the workspace. (k_kv_attn_keys counts arrivals there too.)
static int64_t kv_held(const KvShape &s, int variant, int64_t wgs) {
  if (variant < 2 && wgs * 4 > kKvArrivalBytes) return 1;
  const int64_t held = s.part_rows / kv_variant_rows(variant) / wgs;
  return held < 1 ? 1 : held < 256 ? held : 256;
}

// The plan of a variant: the number of key splits that takes the least time by these figures, in us as measured (MI355X).
// - k_kv_attn_keys: a workgroup takes a step of 32 keys in (0.08 + 0.0011 D) WR us when it is not held up by the others
//   (one sequence of 131072 keys, 8 heads of 128: 8 splits 83 us, 16 splits 48, 32 splits 46 = 5.9 TB/s), together they
//   take 1 / 5.5 TB/s, not quite hiding one under the other, and the last one joins its tile's splits at about 1 us a
//   round trip (192 splits of 4 rows: 71 us against 46). 48 sequences of 2 k to 8 k keys: 1 split 114 us, 2 110, 4 105, 8 109.
// - k_kv_attn_rows: a step of 32 keys takes 0.24 + 0.0028 D us alone on a CU and no less than 0.04 + 0.0023 D for each
//   workgroup of a CU that runs one; two terms 1.22 and 1.39 times that, 128 rows 1.22 and 1.68 times. A workgroup's rows
//   and results cost about 6 steps. Joining takes 4 us and the partial results' way to memory and back. (512 tokens
//   behind 7680, 32 / 8 heads, D = 128 in 64 rows: 1 split 150 us, 2 114, 4 100, 8 107. Over 200 measured times of D = 64
//   to 256 the figures are off by 10 % rms, and the number that they choose costs at most 13 % more than the best.)
static KvPlan kv_plan_variant(const KvShape &s, int variant) {
  const int64_t R = kv_variant_rows(variant), cus = device_cu_count();
  const int64_t units = variant < 2 ? s.B : s.T * s.G / R + s.B, held = kv_held(s, variant, units * s.Hkv);
  // workgroups that have keys: sequences of equal length
  const int64_t even = (s.T + s.B - 1) / s.B * s.G;
  const int64_t wgs = (variant < 2 ? s.B : s.B * ((even + R - 1) / R)) * s.Hkv;
  const int64_t keys = kv_keys(s, R), steps = (keys + 31) / 32;
  const int64_t rows = s.new_rows * s.G < R ? s.new_rows * s.G : R;
  const double alone = variant < 2 ? (0.08 + 0.0011 * s.D) * (R / 16)
                                   : (0.24 + 0.0028 * s.D) * (s.two ? 1.22 : 1.0) * (R == 128 ? 1.22 : 1.0);
  const double share = (0.04 + 0.0023 * s.D) * (s.two ? 1.39 : 1.0) * (R == 128 ? 1.68 : 1.0);
  // of the most keys, how many a workgroup sees on average
  const double seen = !s.causal || s.window ? 1.0 : s.new_rows < keys ? 1.0 - 0.5 * s.new_rows / keys : 0.5;
  const int64_t items = rows * (s.D / 4);
  auto join = [&](int64_t n) {  // round trips of the last workgroup
    return items <= 512 ? 1 + 0.7 * ((n + 7) / 8) * ((items + 255) / 256) : 4 + 1.0 * ((n + 3) / 4) * ((items + 1023) / 1024);
  };
  auto time_of = [&](int64_t n) {
    const double mine = static_cast<double>(steps) / n;
    if (variant < 2) {
      const int64_t slots = cus * (s.D <= 128 ? 2 : 1);
      const double own = alone * mine * ((wgs * n + slots - 1) / slots), read = static_cast<double>(wgs) * steps * 64 * s.D / 5.5e6;
      return (own > read ? own : read) + 0.3 * own + (n > 1 ? join(n) : 0);
    }
    const double one = (mine + 6) * alone, all = (mine * seen + 6) * share * ((wgs * n + cus - 1) / cus);
    return sqrt(sqrt(one * one * one * one + all * all * all * all)) + (n > 1 ? 4 + 1.2e-6 * wgs * n * R * (s.D + 2) : 0);
  };
  const int64_t least = (keys + kKvSplitKeys - 1) / kKvSplitKeys;
  KvPlan p{variant, units, least < held ? least : held, 0, false};
  if (const char *e = tuning_env("VYBDQ_KV_SPLITS")) {
    const int64_t n = atoi(e) < 0 ? -atoi(e) : atoi(e);
    p.splits = n < 1 ? 1 : n < held ? n : held;
    p.time = time_of(p.splits);
    p.by_length = atoi(e) < 0 && variant < 2 && s.B > 1 && s.B <= 64 && p.splits > 1;
    return p;
  }
  p.time = time_of(p.splits);
  for (int64_t n = p.splits + 1; n <= held && 4 * n <= steps; n += 1 + n / 16) {  // (some 60 numbers at most: this is host time)
    const double time = time_of(n);
    if (time < p.time) {
      p.time = time;
      p.splits = n;
    }
  }
  // By length where the call is long enough to gain by it (more than 64 sequences are many workgroups already). Sequences of
  // one to the full length, us with and without: 12 of 6000 tokens, 4 heads of 128: 16.2, 15.1; of 256, 2 rows: 26.9, 27.6, 5
  // rows 38.1, 42.0; 48 of 8192, 8 heads of 128: 101.3, 104.4; 4 of 131072: 131, 142. (All of full length: 34.6, 33.0 and
  // 55.2, 54.3.)
  p.by_length = variant < 2 && s.B > 1 && s.B <= 64 && p.splits > 1 && p.time >= 25;
  return p;
}

// Variant by the rows that share keys. Up to 16 (a decode step): k_kv_attn_keys, whose waves need not wait for each other. 17
// to 32 (drafted tokens): the same, but for few sequences of many keys, whose last workgroups would be long in joining
// 32 rows; k_kv_attn_rows joins them in a launch of its own (8 rows of 4 heads, 8 key heads of 128, bf16, us of the one and
// the other: 1 sequence of 300 keys 9.9, 11.9, of 2000 15.3, 12.3, of 12000 25.6, 19.2; 3 of 2000 20.0, 15.5, of 12000 31.8,
// 34.0; 8 of 2000 20.7, 19.9, of 12000 43.7, 49.9; 20 of 12000 112, 130: the rule takes the slower one at 8 of 2000, by 4 %, and
// stands on these eight for other head sizes and float32 queries too). More: k_kv_attn_rows, whose waves share the
// conversion (16 sequences of 6000 keys, 64 rows: 78 us against 147). Its tiles of 128 rows need half the cache reads, those
// of 64 keep more waves and even out better: 128 rows only where D = 128 leaves room for their registers and the figures
// above give them the lesser time (512 tokens behind 7680: 93 us against 103; a prompt of 2048: 64 against 57).
static KvPlan kv_plan(const KvShape &s) {
  const int64_t rows = s.new_rows * s.G;
  const bool wide = s.D == 128 && !s.two;
  if (const char *e = tuning_env("VYBDQ_KV_VARIANT")) {
    const int v = atoi(e);
    if (v >= 0 && v < (wide ? kKvVariants : kKvVariants - 1)) return kv_plan_variant(s, v);
  }
  const int64_t steps = (kv_keys(s, 32) + 31) / 32;
  if (rows <= 16) return kv_plan_variant(s, 0);
  if (rows <= 32 && (steps < 60 || s.B * s.Hkv * steps > 3500)) return kv_plan_variant(s, 1);
  const KvPlan p = kv_plan_variant(s, 2);
  if (!wide) return p;
  const KvPlan q = kv_plan_variant(s, 3);
  return q.time < p.time ? q : p;
}

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
  VYBDQ_REQUIRE(T * Hq < (int64_t(1) << 31), VYBDQ_ERR_SHAPE, "T * Hq must be below 2^31");
  VYBDQ_REQUIRE(W >= 1 && W * page < (int64_t(1) << 30), VYBDQ_ERR_SHAPE, "W must be at least 1 and W * page below 2^30");
  VYBDQ_REQUIRE(window >= 0 && window < (int64_t(1) << 30), VYBDQ_ERR_SHAPE, "window must be in 0 .. 2^30 - 1");
  // (a grid holds less than 2^32 threads along x)
  VYBDQ_REQUIRE((T * (Hq / Hkv) / 64 + B) * Hkv < (int64_t(1) << 24), VYBDQ_ERR_SHAPE, "(T Hq / (64 Hkv) + B) Hkv must be below 2^24");
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
  const int64_t cap = W * page, tokens = max_ctx >= 1 && max_ctx < cap ? max_ctx : cap;
  const int64_t most = max_new >= 1 && max_new < T ? max_new : T;
  const KvShape shape{D, Hkv, G, T, B, most, tokens, two, causal != 0, window,
                      ws && ws_bytes > kKvArrivalBytes ? (ws_bytes - kKvArrivalBytes) / ((D + 2) * 4) : 0};
  const KvPlan plan = kv_plan(shape);
  VYBDQ_REQUIRE(kv_keys(shape, kv_variant_rows(plan.variant)) <= plan.splits * kKvSplitKeys, VYBDQ_ERR_SHAPE,
                "more than 2^24 keys of a row to a split (of max_ctx, or of W * page): the workspace is too small to split them");
  KvAttnArgs a{};
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
  a.splits = static_cast<int32_t>(plan.splits);
  a.by_length = plan.by_length;
  const dim3 grid(static_cast<unsigned>(plan.units * Hkv * (plan.variant < 2 ? plan.splits : 1)),
                  static_cast<unsigned>(plan.variant < 2 ? 1 : plan.splits));
  if (two) kv_attn_launch_f(static_cast<int>(D), plan.variant, a, grid, as_stream(stream));
  else kv_attn_launch_h(static_cast<int>(D), plan.variant, a, grid, as_stream(stream));
  return check_launch("vybdq_kv_attn");
}
