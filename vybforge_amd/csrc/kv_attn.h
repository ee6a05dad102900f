// Attention over the paged 8-bit cache (layout: kv.h), gfx950: from single tokens of many sequences to prompt
// chunks, grouped heads, causal, with or without a sliding window.
//
//   t_ij = (q_i . k_j) scale log2(e) 2^ek + ev     (ek, ev: exponents of key j's page for K and V)
//   w_ij = 2^(t_ij - m_i), acc_i = sum_j w_ij v_j, l_i = sum_j w_ij 2^-ev, o_i = acc_i / l_i
// with v_j, k_j the bare codes: the K scale is one factor per 16 keys in the exponent's fma, and the V scale rides
// in the exponent too, so no code is ever multiplied by its scale. m_i is a running reference that follows the
// largest t: w stays within 2^15, whatever the pages' scales are (references from 2^22 on: kKvFar below). One pass over the keys.
//
// Matrix instructions (16x16x32 fp16, float32 sums) on transposed products, so that nothing is ever moved between
// lanes: S^T = K Q^T puts 4 consecutive keys of one query row in a lane, and that is already the layout in which
// O^T = V^T P^T wants P^T, the order of the 32 keys within an instruction being free. K and V codes go from the
// cache straight into operand registers (16-byte loads, one e4m3 -> fp16 conversion per two codes; every e4m3
// value is an fp16 value). Rounded to fp16: the query row, scaled by the power of two that brings its largest
// value into [2^14, 2^15) (exact for fp16 values, and for bf16 ones down to 2^-31 of the largest; below that off by 2^-39 of it
// at most), and w (11 bits down to 2^-22 of the row's largest). For float32 queries both are split into two fp16 terms (22 bits).
//
// A wave owns 16 NCT query rows (row = token * G + head of the group; the G query heads of a key head read the
// same keys, so they share its tiles) and takes 32 keys at a step. Few rows: k_kv_attn_keys, whose waves take turns over the
// keys; more: k_kv_attn_rows, whose waves own rows each and share the keys. Where the rows alone leave the chip idle the keys
// are split over workgroups too: each stores its (m, l, acc), and they are joined in split order, so results do
// not depend on the order of arrival.
//
// What bounds them, MI355X (a large copy runs at 4.7 TB/s, a large fp16 product at 1089 TFLOP/s): 48 sequences of 2 to 8 k
// tokens, one row each, 32 / 8 heads of 128: 101 us, 5.1 TB/s of codes; 4 of up to 131072: 132 us, 5.5 TB/s. A prompt of 4096
// tokens: 165 us, 831 TFLOP/s; 513 tokens behind 32 k: 331 us, 825 TFLOP/s. Of the prompt's time the matrix instructions
// (18 cycles each on a SIMD with four waves) are 64 us, the LDS reads that feed them 30 (128 rows) to 60 (64 rows) beside
// them; when it took 180, it took 141 without loads and conversion and 169 without exponentials. With heads of 64 a step
// of 16 rows is 130 cycles of matrix instructions and some 310 of vector instructions, two thirds of them the softmax: 464
// TFLOP/s with a window of 4096. 32x32x16 instructions in the same scheme were no faster (prompt 177 to 188 us, heads of
// 64 83 to 97 against 87), nor were two tiles of 16 rows of heads of 64 to a wave (93 against 87).
#pragma once

#include "kv.h"

#include <type_traits>

namespace vybdq {

struct KvAttnArgs {
  KvCacheArgs c;
  KvBatchArgs b;
  const void *q;
  void *out;
  float *lse;
  uint32_t *arrivals;  // per (tile, head): zero between calls
  float *part;         // per (tile, head, split): m [R], l [R], acc [R][D]
  int64_t ldq;
  int32_t G, dt;       // dt: F32, F16 or BF16 of q and out
  int32_t causal, window;
  float scale2;        // scale * log2(e)
  int32_t splits;      // k_kv_attn_keys: workgroups of a sequence and head, on average
  int32_t by_length;   // and whether a sequence's number of them goes with its length
};

// Four e4m3 codes as fp16 (exact).
__device__ __forceinline__ void kv_dec4(uint32_t w, h2 &a, h2 &b) {
  a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false);
  b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true);
}

__device__ __forceinline__ h8 kv_dec8(uint32_t lo, uint32_t hi) {
  h2 a, b, c, d;
  kv_dec4(lo, a, b);
  kv_dec4(hi, c, d);
  return h8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// over the four lanes that hold one query row (lanes l, l ^ 16, l ^ 32, l ^ 48)
__device__ __forceinline__ float col_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float col_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// 16 consecutive elements of a row as float32. TWO: float32 elements, else fp16 or bf16.
template <bool TWO>
__device__ __forceinline__ void load16(const void *p, bool bf16, int64_t i, float (&x)[16]) {
  if constexpr (TWO) {
    const f4 *s = reinterpret_cast<const f4 *>(static_cast<const float *>(p) + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f4 v = s[j];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * j + e] = v[e];
    }
  } else {
    const u4 *s = reinterpret_cast<const u4 *>(static_cast<const uint16_t *>(p) + i);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const u4 v = s[j];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t w = v[e];
        const float h0 = half_bits_to_f32(w & 0xffffu), h1 = half_bits_to_f32(w >> 16);
        x[8 * j + 2 * e] = bf16 ? __uint_as_float(w << 16) : h0;
        x[8 * j + 2 * e + 1] = bf16 ? __uint_as_float(w & 0xffff0000u) : h1;
      }
    }
  }
}

// N consecutive outputs (N even), rounded once to the output type
template <bool TWO, int N>
__device__ __forceinline__ void store_n(void *p, bool bf16, int64_t i, const float (&x)[N]) {
  if constexpr (TWO) {
    f2 *o = reinterpret_cast<f2 *>(static_cast<float *>(p) + i);
#pragma unroll
    for (int j = 0; j < N / 2; ++j) o[j] = f2{x[2 * j], x[2 * j + 1]};
  } else {
    uint32_t *o = reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(p) + i);
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
      const uint32_t b = f32_to_bf16(x[2 * j]) | (static_cast<uint32_t>(f32_to_bf16(x[2 * j + 1])) << 16);
      const h2 f = {static_cast<_Float16>(x[2 * j]), static_cast<_Float16>(x[2 * j + 1])};
      o[j] = bf16 ? b : __builtin_bit_cast(uint32_t, f);
    }
  }
}

// Variants. 0, 1: k_kv_attn_keys, 16 or 32 query rows to a workgroup; 2, 3: k_kv_attn_rows, 64 or 128.
constexpr int kKvVariants = 4;
constexpr int kv_variant_rows(int variant) { return variant == 0 ? 16 : variant == 1 ? 32 : variant == 2 ? 64 : 128; }

// A row's reference is 2^-8 of its largest weight, or up to twice that, when it is taken, and is taken anew once a weight would
// pass 2^15: weights as fp16 operands then hold all their bits down to 2^-22 of the largest and vanish below 2^-33. It is a
// whole number, so that it adds to a V scale's exponent without rounding, and no larger, because exponents from 8 on are
// rounded to 2^-21. With two terms (float32 queries) the reference is the largest weight, and the 2^12 that two terms
// need are a product behind the exponential: 22 bits down to 2^-15 of the largest, below that 2^-37 of it. (lse, relative, of
// 4 keys and float32 queries: 1.9e-7, with the 2^12 in the exponent 4.7e-7; of 34 keys and bf16 ones with 2^12: 2.3e-7.)
constexpr float kv_ref(bool two) { return two ? 0.0f : 8.0f; }
constexpr float kv_move(bool two) { return two ? 3.0f : 15.0f; }
constexpr float kv_lift(bool two) { return two ? 4096.0f : 1.0f; }
constexpr float kKvNone = -3.402823466e38f;  // the reference of a row that has seen nothing: the lowest finite (no inf - inf)
#define KV_NEG_INF (-__builtin_inff())

// From references of 2^22 on (scores times log2 e) float32 no longer holds a score and a V scale's exponent side by side, nor
// what is left of a product beside its rounded self: t - m, rounded other than m was, could leave a weight at 2^64 or at nothing.
// A wave one of whose rows gets there keeps the two apart from then on: weight 2^((p - m) + (ev - scale)), with p the product
// rounded to float32, m the largest p of the row, and scale, one number for the wave, 2^-8 of the largest V scale so far (two
// terms: that scale). Equal products then have equal weights of whatever size they are, and none is above 2^8. The price is that
// V scales count against each other over a whole wave: weights of pages 2^22 (two terms: 2^15) below the largest lose bits.
constexpr float kKvFar = 4194304.0f;
struct KvFar {
  float limit;  // kv_move(), or NaN in a wave that is there: every step then takes the branch that moves references
  float scale;
};

// What the kernels only read, through the constant address space: uniform reads become scalar loads.
template <class T>
__device__ __forceinline__ T kv_const(const T *p, int64_t i) {
  return ((const T __attribute__((address_space(4))) *)p)[i];
}

// A tile of query rows: rows r0 .. of sequence b's n G (row = token * G + head of the group), and its keys.
struct KvTile {
  KvSeq sq;
  int rows, r0;        // (T G < 2^31)
  int ctx, p0;         // tokens; position of the first row
  int k0, steps;       // keys that some row of the tile sees lie in k0 .. k0 + 32 steps - 1
  int free0, free1;    // keys that every row sees: no mask
  const int32_t *table;
  bool past;           // tokens past the table's pages: the rows are NaN
};

__device__ __forceinline__ bool kv_tile_seq(const KvAttnArgs &a, int b, KvTile &t) {
  t.sq = kv_seq(a.b, b);
  t.rows = t.sq.n * a.G;
  t.past = t.sq.ctx > (a.b.W << a.c.ps);
  if (t.past && (threadIdx.x & 63) == 0) kv_flag(a.b.status, kKvBadCtx);
  t.ctx = t.sq.ctx > 0 && !t.past ? t.sq.ctx : 0;
  t.p0 = t.ctx - t.sq.n;
  t.table = a.b.table + static_cast<int64_t>(b) * a.b.W;
  return t.rows > 0;
}

// Tile u of the batch. Sequence b's tiles are units first(b) ..: ceil(n G / R) of them, and
// floor((s + n) G / R) - floor(s G / R) + 1 is no less.
__device__ __forceinline__ bool kv_tile_unit(const KvAttnArgs &a, int R, int u, KvTile &t) {
  auto first = [&](int i) { return static_cast<int64_t>(static_cast<uint32_t>(a.b.q_start[i]) * static_cast<uint32_t>(a.G) / R + i); };
  const int b = kv_find(a.b.B, u, first);
  const int64_t r0 = (u - first(b)) * R;
  t.r0 = static_cast<int>(r0 < a.b.T * a.G ? r0 : -1);
  return t.r0 >= 0 && kv_tile_seq(a, b, t) && t.r0 < t.rows;
}

__device__ __forceinline__ void kv_tile_keys(const KvAttnArgs &a, int R, KvTile &t) {
  const int i_lo = t.r0 / a.G, i_hi = ((t.rows - t.r0 > R ? t.r0 + R : t.rows) - 1) / a.G;
  int k1 = a.causal ? t.p0 + i_hi + 1 : t.ctx;
  k1 = k1 > 0 ? k1 : 0;
  const int first = a.window ? t.p0 + i_lo - a.window + 1 : 0;
  t.k0 = (first > 0 ? first : 0) & ~15;  // (whole blocks of 16: the pages before them may be gone)
  t.steps = k1 > t.k0 ? (k1 - t.k0 + 31) >> 5 : 0;
  t.free0 = a.window ? t.p0 + i_hi - a.window + 1 : 0;
  t.free1 = a.causal ? t.p0 + i_lo + 1 : t.ctx;
}

// The first step of split i of S. (No product of steps and splits: 2^25 steps in 256 splits pass 32 bits.)
__device__ __forceinline__ int kv_split(int steps, int i, int S) {
  const int rest = steps % S;
  return steps / S * i + (i < rest ? i : rest);
}

// The sum over this lane and those below it.
template <class T>
__device__ __forceinline__ T lane_scan(T v) {
  auto from = [&](auto ctrl, auto rows) {
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(ctrl)::value, decltype(rows)::value, 0xf, false));
  };
  using std::integral_constant;
  v += from(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});  // row_shr 1, 2, 4, 8: rows of 16
  v += from(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
  v += from(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
  v += from(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
  v += from(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});  // row_bcast 15: into rows 1 and 3
  v += from(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});  // row_bcast 31: into rows 2 and 3
  return v;
}

// Which sequence and part of its keys unit u of k_kv_attn_keys takes. There are B a.splits units for each head. By length (B up
// to 64, a lane each), a sequence has a number of them that goes with its own keys (those of its first tile, in steps of 32),
// so that sequences of unequal lengths end together: the largest share, of four tried, whose parts fit in the units. Every
// workgroup finds the same numbers. That costs 1 us at its start, and the longest sequence's join takes longer.
struct KvPart {
  int b, split, S;
};
__device__ __forceinline__ KvPart kv_part(const KvAttnArgs &a, int R, int u) {
  const int B = a.b.B, S = a.splits;
  if (!a.by_length) return {u / S, u % S, S};
  const int b = threadIdx.x & 63;
  float steps = 0.f;
  if (b < B) {
    const int s0 = a.b.q_start[b], s1 = a.b.q_start[b + 1], ctx = a.b.ctx[b];
    if (s0 >= 0 && s0 < s1 && s1 <= a.b.T && ctx > 0 && ctx <= (a.b.W << a.c.ps)) {
      KvTile t;
      t.rows = (s1 - s0) * a.G;
      t.r0 = 0;
      t.ctx = ctx;
      t.p0 = ctx - (s1 - s0);
      kv_tile_keys(a, R, t);
      steps = static_cast<float>(t.steps);
    }
  }
  const float total = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(lane_scan(steps)), 63));
  // parts per step: units / total, and less, down to what fits whatever is rounded up: sum of ceil(x) < sum of x + B
  const float inv = total > 0.f ? B / total : 0.f;
  int mine = b < B ? 1 : 0, upto = b < B ? b + 1 : B;  // (one part each, should rounding ever leave none that fits)
#pragma unroll
  for (int k = 3; k >= 0; --k) {
    const int n = static_cast<int>(ceilf(steps * fminf((S - k * (1.f / 3)) * inv, 0.25f)));
    const int parts = b < B ? (n > 1 ? n : 1) : 0, sum = lane_scan(parts);
    if (__builtin_amdgcn_readlane(sum, 63) <= B * S) {
      mine = parts;
      upto = sum;
    }
  }
  const int owner = __popcll(__ballot(upto <= u));
  if (owner >= 64) return {-1, 0, 1};  // (a unit that no sequence has)
  return {owner, u - __builtin_amdgcn_readlane(upto - mine, owner), __builtin_amdgcn_readlane(mine, owner)};
}

// The 16 query rows r .. r + 15 as operands of S^T = K Q^T, one row per column: lane (col, g4) holds dims
// 64 c + 16 g4 + 8 x + 0 .. 7 in f[2 c + x], scaled by the power of two that brings the row's largest value
// into [2^14, 2^15). qc: the factor from their products with K codes to scale * log2(e) q . (K code).
template <int C, bool TWO>
struct KvRows {
  h8 f[2 * C][TWO ? 2 : 1];
  float qc;
  int lo, hi;  // keys lo .. hi - 1 are seen
};

template <int C, bool TWO>
__device__ __forceinline__ void kv_load_rows(const KvAttnArgs &a, const KvTile &t, int r, int h, KvRows<C, TWO> &q) {
  constexpr int D = 64 * C;
  const int lane = threadIdx.x & 63, g4 = lane >> 4;
  r += lane & 15;
  const bool have = r < t.rows;
  // (places past the last row: its values, not stored; a row of this tile, which no other workgroup writes where out is q)
  const int rr = have ? r : t.rows - 1;
  const int i = rr / a.G, hq = h * a.G + rr % a.G;
  q.hi = !have ? 0 : a.causal ? t.p0 + i + 1 : t.ctx;
  q.lo = a.window ? t.p0 + i - a.window + 1 : 0;
  const int64_t at = (t.sq.s0 + i) * a.ldq + hq * D + 16 * g4;
  const bool bf16 = a.dt == VYBDQ_BF16;
  float x[C][16], amax = 0.f;
  bool bad = false;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    load16<TWO>(a.q, bf16, at + 64 * c, x[c]);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      bad |= (__float_as_uint(x[c][e]) & 0x7fffffffu) >= 0x7f800000u;
      amax = fmaxf(amax, fabsf(x[c][e]));
    }
  }
  float inv;
  const float sc = block_scale(col_max(amax), inv);
  // an infinity or NaN in any of the row's four lanes makes its scores NaN
  q.qc = sc * a.scale2 + col_sum(bad ? __builtin_nanf("") : 0.f);
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float v = x[c][e] * inv;
      const _Float16 f = static_cast<_Float16>(v);
      q.f[2 * c + e / 8][0][e % 8] = f;
      if constexpr (TWO) q.f[2 * c + e / 8][1][e % 8] = static_cast<_Float16>(v - static_cast<float>(f));
    }
}

__device__ __forceinline__ float kv_uniform(float x) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(x))); }

// Weights of one tile of scores. s[ct][n]: the products of 2 blocks of 16 keys with the rows of column tile ct; ks, ev, iv: the
// blocks' K scale, V exponent and 2^-ev. Updates m, far, l and acc, returns the weights as operands of O^T = V^T P^T.
template <int NCT, int C, bool TWO>
__device__ __forceinline__ void kv_weights(const f4 (&s)[NCT][2], const KvRows<C, TWO> (&q)[NCT], const float (&ks)[2],
                                           const float (&ev)[2], const float (&iv)[2], int tok, bool masked, KvFar &far,
                                           float (&m)[NCT], float (&l)[NCT], f4 (&acc)[NCT][4 * C], h8 (&p)[NCT][TWO ? 2 : 1]) {
  const int g4 = (threadIdx.x & 63) >> 4;
  float t[NCT][8];
  auto hide = [&]() {
#pragma unroll
    for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = tok + 16 * n + 4 * g4 + e;
          t[ct][4 * n + e] = key >= q[ct].lo && key < q[ct].hi ? t[ct][4 * n + e] : KV_NEG_INF;
        }
  };
  auto exponents = [&]() {  // t - m
#pragma unroll
    for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float ck = q[ct].qc * ks[n], add = ev[n] - m[ct];
#pragma unroll
        for (int e = 0; e < 4; ++e) t[ct][4 * n + e] = __builtin_fmaf(s[ct][n][e], ck, add);
      }
    if (masked) hide();
  };
  exponents();
  float top[NCT], any = KV_NEG_INF;
#pragma unroll
  for (int ct = 0; ct < NCT; ++ct) {
    top[ct] = t[ct][0];
#pragma unroll
    for (int e = 1; e < 8; ++e) top[ct] = fmaxf(top[ct], t[ct][e]);
    any = fmaxf(any, top[ct]);
  }
  // (told to be rare: laid out as likely ones, the two branches cost a prompt 3 %)
  if (__builtin_expect(__ballot(!(any <= far.limit)) != 0, 0)) {
    if (__builtin_expect(far.limit == kv_move(TWO), 1)) {
      float now[NCT];
      bool beyond = false;
#pragma unroll
      for (int ct = 0; ct < NCT; ++ct) {
        // the largest exponent itself, not its difference to the old reference (which may be kKvNone)
        float big = KV_NEG_INF;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            big = fmaxf(big, t[ct][4 * n + e] == KV_NEG_INF ? KV_NEG_INF : __builtin_fmaf(s[ct][n][e], q[ct].qc * ks[n], ev[n]));
        now[ct] = fmaxf(m[ct], ceilf(col_max(big)) - kv_ref(TWO));
        beyond |= fabsf(now[ct]) >= kKvFar && now[ct] != kKvNone;
      }
      if (__ballot(beyond)) {
        far = {__builtin_nanf(""), kv_uniform(fmaxf(ev[0], ev[1]) - kv_ref(TWO))};
#pragma unroll
        for (int ct = 0; ct < NCT; ++ct) m[ct] -= far.scale;
      } else {
#pragma unroll
        for (int ct = 0; ct < NCT; ++ct) {
          const float f = __builtin_amdgcn_exp2f(m[ct] - now[ct]);
          m[ct] = now[ct];
          l[ct] *= f;
#pragma unroll
          for (int d = 0; d < 4 * C; ++d) acc[ct][d] *= f;
        }
        exponents();
      }
    }
    if (far.limit != kv_move(TWO)) {
#pragma clang fp contract(off)
      const float scale = kv_uniform(fmaxf(far.scale, fmaxf(ev[0], ev[1]) - kv_ref(TWO)));
#pragma unroll
      for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float ck = q[ct].qc * ks[n];
#pragma unroll
          for (int e = 0; e < 4; ++e) t[ct][4 * n + e] = s[ct][n][e] * ck;
        }
      if (masked) hide();
#pragma unroll
      for (int ct = 0; ct < NCT; ++ct) {
        float big = t[ct][0];
#pragma unroll
        for (int e = 1; e < 8; ++e) big = fmaxf(big, t[ct][e]);
        big = col_max(big);
        // (whole numbers where they can be, as elsewhere: p - m is then rounded once)
        const float now = fmaxf(m[ct], fabsf(big) < kKvFar ? ceilf(big) : big);
        const float f = __builtin_amdgcn_exp2f((m[ct] - now) + (far.scale - scale));
        m[ct] = now;
        l[ct] *= f;
#pragma unroll
        for (int d = 0; d < 4 * C; ++d) acc[ct][d] *= f;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) t[ct][4 * n + e] = (t[ct][4 * n + e] - now) + (ev[n] - scale);
      }
      far.scale = scale;
    }
  }
#pragma unroll
  for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      float w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = __builtin_amdgcn_exp2f(t[ct][4 * n + e]);
      // not of the rounded weights: lse is a float32 result
      l[ct] = __builtin_fmaf((w[0] + w[1]) + (w[2] + w[3]), iv[n], l[ct]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = w[e] * kv_lift(TWO);
        const _Float16 f = static_cast<_Float16>(x);
        p[ct][0][4 * n + e] = f;
        if constexpr (TWO) p[ct][1][4 * n + e] = static_cast<_Float16>(x - static_cast<float>(f));
      }
    }
}

// A wave's sums as every other's: m alone their reference. It stays the row's p where that is far, so that equal products are
// joined with equal weights.
template <int NCT, int C, bool TWO>
__device__ __forceinline__ void kv_settle(const KvFar &far, float (&m)[NCT], float (&l)[NCT], f4 (&acc)[NCT][4 * C]) {
  if (far.limit == kv_move(TWO)) return;
#pragma unroll
  for (int ct = 0; ct < NCT; ++ct) {
    const float r = fabsf(m[ct]) < kKvFar ? kv_ref(TWO) : 0.f, f = __builtin_amdgcn_exp2f(far.scale + r);
    m[ct] -= r;
    l[ct] *= f;
#pragma unroll
    for (int d = 0; d < 4 * C; ++d) acc[ct][d] *= f;
  }
}

// Where a tile's results go: the output, or the workspace as one of S partial results. COHERENT: partials that another
// workgroup of the same launch reads (stored through the XCD's L2), else plain stores for the next launch.
template <int D, int R, bool TWO, bool COHERENT>
struct KvSink {
  const KvAttnArgs &a;
  const KvTile &t;
  int h;
  bool whole;
  float *part;  // this split's: m, l interleaved [R], acc [R][D]

  // N dims d .. of tile row r: sums x over weights of sum lr, reference mr
  template <int N>
  __device__ __forceinline__ void finish(int r, float mr, float lr, int d, const float (&x)[N]) const {
    const int rr = t.r0 + r;
    if (rr >= t.rows) return;
    const int64_t at = (t.sq.s0 + rr / a.G) * (static_cast<int64_t>(a.c.Hkv) * a.G) + h * a.G + rr % a.G;
    const float f = lr == 0.f ? 0.f : (1.0f / kv_lift(TWO)) / lr;
    float y[N];
#pragma unroll
    for (int e = 0; e < N; ++e) y[e] = x[e] * f;
    store_n<TWO, N>(a.out, a.dt == VYBDQ_BF16, at * D + d, y);
    if (a.lse && d == 0) {  // ln 2 (m + log2 l), the logarithm of a number near one, ln 2 as a float32 and the rest of it
      constexpr double kLn2 = 0.6931471805599453;
      constexpr float hi = static_cast<float>(kLn2), lo = static_cast<float>(kLn2 - hi), r = kv_ref(TWO);
      const float at_max = mr + r, rest = __builtin_amdgcn_logf(lr * (TWO ? 1.0f : 1.0f / 256));
      a.lse[at] = lr == 0.f ? KV_NEG_INF : __builtin_fmaf(at_max, hi, __builtin_fmaf(rest, hi, at_max * lo));
    }
  }
  template <int N>
  __device__ __forceinline__ void put(int r, float mr, float lr, int d, const float (&x)[N]) const {
    if (whole) {
      finish<N>(r, mr, lr, d, x);
    } else if (t.r0 + r < t.rows && !COHERENT) {
      f2 *o = reinterpret_cast<f2 *>(part + 2 * R + r * D + d);
#pragma unroll
      for (int e = 0; e < N / 2; ++e) o[e] = f2{x[2 * e], x[2 * e + 1]};
      if (d == 0) reinterpret_cast<f2 *>(part)[r] = f2{mr, lr};
    } else if (t.r0 + r < t.rows) {
      uint64_t *o = reinterpret_cast<uint64_t *>(part + 2 * R + r * D + d);
#pragma unroll
      for (int e = 0; e < N / 2; ++e)
        __hip_atomic_store(o + e, __float_as_uint(x[2 * e]) | (static_cast<uint64_t>(__float_as_uint(x[2 * e + 1])) << 32),
                           __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (d == 0)
        __hip_atomic_store(reinterpret_cast<uint64_t *>(part) + r,
                           __float_as_uint(mr) | (static_cast<uint64_t>(__float_as_uint(lr)) << 32), __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
    }
  }

  static __device__ __forceinline__ f2 load_through(const float *p) {
    return __builtin_bit_cast(f2, __hip_atomic_load(reinterpret_cast<const uint64_t *>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
  }

  // Items it, it + step, .. (N of them, those before `items`) of a tile's rows from S splits' results at `all`, `stride` floats apart: item i is 4 dims
  // of a row. Joined in split order, with N W splits' loads to a round trip. THROUGH: read past the caches, 8 bytes at a time.
  template <int N, int W, bool THROUGH>
  __device__ __forceinline__ void finish_joined(const float *all, int64_t stride, int S, int it, int step, int items) const {
    int r[N], d[N];
    float mr[N], lr[N], x[N][4];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = it + i * step < items ? it + i * step : it;
      r[i] = at / (D / 4);
      d[i] = at % (D / 4) * 4;
      mr[i] = kKvNone;
      lr[i] = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[i][e] = 0.f;
    }
#pragma unroll 1
    for (int w0 = 0; w0 < S; w0 += W) {
      f2 ml[N][W];
      f4 v[N][W];
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const float *pw = all + (w0 + w < S ? w0 + w : S - 1) * stride;
          const float *pv = pw + 2 * R + r[i] * D + d[i];
          if constexpr (THROUGH) {
            ml[i][w] = load_through(pw + 2 * r[i]);
            const f2 lo = load_through(pv), hi = load_through(pv + 2);
            v[i][w] = f4{lo.x, lo.y, hi.x, hi.y};
          } else {
            ml[i][w] = reinterpret_cast<const f2 *>(pw)[r[i]];
            v[i][w] = *reinterpret_cast<const f4 *>(pv);
          }
        }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float now = mr[i];
#pragma unroll
        for (int w = 0; w < W; ++w)
          if (w0 + w < S) now = fmaxf(now, ml[i][w].x);
        const float f0 = __builtin_amdgcn_exp2f(mr[i] - now);
        mr[i] = now;
        lr[i] *= f0;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[i][e] *= f0;
#pragma unroll
        for (int w = 0; w < W; ++w)
          if (w0 + w < S) {
            const float f = __builtin_amdgcn_exp2f(ml[i][w].x - now);
            lr[i] = __builtin_fmaf(f, ml[i][w].y, lr[i]);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[i][e] = __builtin_fmaf(f, v[i][w][e], x[i][e]);
          }
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (it + i * step < items) finish<4>(r[i], mr[i], lr[i], d[i], x[i]);
  }

  // All S splits' results of the tile, joined by the last workgroup to arrive. They are stored through the XCD's L2 and
  // have completed before the arrival is counted. Few are read past the caches; for many, what the caches hold of them is
  // dropped first, 1 us that 16-byte reads make good (5 splits, 30 rows of 256 dims: 44.0 us against 46.0 past the caches, 12
  // of 256 33.2 in both, 12 of 128 19.6 past the caches against 20.1, 6 of 128 18.0 against 19.1).
  __device__ __forceinline__ void join(uint32_t *count, int split, int S, bool &is_last) const {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
      const uint32_t old = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      is_last = old == static_cast<uint32_t>(S - 1);
      if (is_last) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!is_last) return;
    const int64_t stride = static_cast<int64_t>(a.c.Hkv) * (R * (D + 2));
    const float *all = part - split * stride;
    const int n_rows = t.rows - t.r0 < R ? t.rows - t.r0 : R, items = n_rows * (D / 4);
    if (items <= 512) {
#pragma unroll 1
      for (int it = threadIdx.x; it < items; it += 256) finish_joined<1, 8, true>(all, stride, S, it, 256, items);
    } else {
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
#pragma unroll 1
      for (int it = threadIdx.x; it < items; it += 1024) finish_joined<4, 4, false>(all, stride, S, it, 256, items);
    }
  }
};

// ---- few rows: the waves of a workgroup take turns over the keys ---------------------------------

// One step of 32 keys on its way: the codes in registers, where the step lies, its blocks' scales.
template <int C>
struct KvStep {
  u4 k[2][C], v[2][C];
  float ks[2], vs[2];
  bool bad[2];
};

// WR groups of 16 rows; the 4 / WR waves of a group take turns over the keys. (The groups' waves read the same codes; the
// second reads come from the CU's own cache.) Two steps of codes in registers leave heads of 192 and 256 one wave a SIMD:
// held to two they spill (64 sequences of 8000 keys, 4 heads of 192: 258 us against 134).
template <int D, int WR, bool TWO>
__global__ void __launch_bounds__(256, D <= 128 ? 2 : 1) k_kv_attn_keys(const KvAttnArgs a) {
  constexpr int C = D / 64, R = 16 * WR, WT = 4 / WR, NQ = TWO ? 2 : 1;
  __shared__ float acc_w[4][16][D + 4];
  __shared__ float ml_w[4][2][16];
  __shared__ bool is_last;
  const int lane = threadIdx.x & 63, col = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wr = wave % WR, wt = wave / WR;
  const int Hkv = a.c.Hkv, h = blockIdx.x % Hkv, ps = a.c.ps, in_page = (1 << ps) - 1;
  const KvPart part = kv_part(a, R, blockIdx.x / Hkv);
  const int split = part.split, S = part.S;
  KvTile t;
  if (part.b < 0 || !kv_tile_seq(a, part.b, t)) return;
  const uint32_t koff = col * D + 16 * g4, voff = 4 * (g4 * D + 4 * col);
  const int last_page = t.ctx > 0 ? (t.ctx - 1) >> ps : 0;

  for (t.r0 = 0; t.r0 < t.rows; t.r0 += R) {
    // a tile beyond the first, which the launch did not plan for, is not split: split 0 takes all its keys
    const bool whole = S == 1 || t.r0 > 0;
    if (whole && split > 0) return;
    kv_tile_keys(a, R, t);
    const int t0 = whole ? 0 : kv_split(t.steps, split, S), t1 = whole ? t.steps : kv_split(t.steps, split + 1, S);

    // pages of a step's two blocks; a block behind the sequence's end takes the last page (its keys are masked)
    auto page_of = [&](int st, int n) {
      const int at = (t.k0 + 32 * st + 16 * n) >> ps;
      return kv_const(t.table, at < last_page ? at : last_page);
    };
    auto fetch = [&](KvStep<C> &x, int st, const int (&pg)[2]) {
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        x.bad[n] = static_cast<uint32_t>(pg[n]) >= static_cast<uint32_t>(a.c.n_pages);
        const int64_t ph = static_cast<int64_t>(x.bad[n] ? 0 : pg[n]) * Hkv + h;
        x.ks[n] = kv_const(a.c.Ks, ph);
        x.vs[n] = kv_const(a.c.Vs, ph);
        const int64_t at = ((ph << ps) + ((t.k0 + 32 * st + 16 * n) & in_page)) * D;
        const uint8_t *kb = a.c.K + at, *vb = a.c.V + at;
#pragma unroll
        for (int c = 0; c < C; ++c) {
          x.k[n][c] = *reinterpret_cast<const u4 *>(kb + (koff + 64 * c));
          x.v[n][c] = *reinterpret_cast<const u4 *>(vb + (voff + 256 * c));
        }
      }
    };

    int st = t0 + wt;
    int pg[2] = {0, 0};
    KvStep<C> even, odd;
    if (st < t1) {
#pragma unroll
      for (int n = 0; n < 2; ++n) pg[n] = page_of(st, n);
      fetch(even, st, pg);
#pragma unroll
      for (int n = 0; n < 2; ++n) pg[n] = page_of(st + WT < t1 ? st + WT : t1 - 1, n);
    }

    KvRows<C, TWO> q[1];
    KvFar far = {kv_move(TWO), 0.f};
    float m[1] = {kKvNone}, l[1] = {t.past ? __builtin_nanf("") : 0.f};
    f4 acc[1][4 * C];
    kv_load_rows<C, TWO>(a, t, t.r0 + 16 * wr, h, q[0]);
#pragma unroll
    for (int d = 0; d < 4 * C; ++d) acc[0][d] = f4{0.f, 0.f, 0.f, 0.f};

    auto use = [&](KvStep<C> &x, int st) {
      const int tok = t.k0 + 32 * st;
      f4 s[1][2];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        s[0][n] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const h8 kf = kv_dec8(x.k[n][c][2 * y], x.k[n][c][2 * y + 1]);
#pragma unroll
            for (int z = 0; z < NQ; ++z) s[0][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, q[0].f[2 * c + y][z], s[0][n], 0, 0, 0);
          }
      }
      float ks[2], ev[2], iv[2];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const uint32_t e = x.bad[n] ? 127u : (__float_as_uint(x.vs[n]) >> 23) & 0xffu;
        ks[n] = x.bad[n] ? __builtin_nanf("") : x.ks[n];
        ev[n] = static_cast<float>(static_cast<int>(e) - 127);
        iv[n] = __uint_as_float((254u - e) << 23);
      }
      // slots behind the sequence's end were never written: their V codes may be anything, NaN included
      if (tok + 32 > t.ctx || x.bad[0] || x.bad[1]) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const int left = x.bad[n] ? 0 : t.ctx - (tok + 16 * n + 4 * g4);
          const uint32_t keep = left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << (8 * left)) - 1;
#pragma unroll
          for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) x.v[n][c][e] &= keep;
          if (x.bad[n] && lane == 0) kv_flag(a.b.status, kKvBadPage);
        }
      }
      h8 p[1][NQ];
      kv_weights<1, C, TWO>(s, q, ks, ev, iv, tok, tok < t.free0 || tok + 32 > t.free1, far, m, l, acc, p);
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const h8 vf = kv_dec8(x.v[0][c][d], x.v[1][c][d]);
#pragma unroll
          for (int z = 0; z < NQ; ++z) acc[0][4 * c + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, p[0][z], acc[0][4 * c + d], 0, 0, 0);
        }
    };

    // two steps to a turn, the next one's codes on their way while one is used, the page numbers one step further ahead (behind
    // the last step they are the last step's again: a load under a condition would have to be waited for where the ways meet)
    auto held = [&](int x) { return x < t1 ? x : t1 - 1; };
    while (st < t1) {
      fetch(odd, held(st + WT), pg);
#pragma unroll
      for (int n = 0; n < 2; ++n) pg[n] = page_of(held(st + 2 * WT), n);
      use(even, st);
      if (st + WT >= t1) break;
      fetch(even, held(st + 2 * WT), pg);
#pragma unroll
      for (int n = 0; n < 2; ++n) pg[n] = page_of(held(st + 3 * WT), n);
      use(odd, st + WT);
      st += 2 * WT;
    }

    // the waves' results, joined through LDS
    const KvSink<D, R, TWO, true> sink{a, t, h, whole, a.part + static_cast<int64_t>(blockIdx.x) * (R * (D + 2))};
    kv_settle<1, C, TWO>(far, m, l, acc);
    l[0] = col_sum(l[0]);
    if (t.r0 > 0) __syncthreads();
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<f4 *>(&acc_w[wave][col][64 * c + 16 * g4 + 4 * e]) =
            f4{acc[0][4 * c][e], acc[0][4 * c + 1][e], acc[0][4 * c + 2][e], acc[0][4 * c + 3][e]};
    if (g4 == 0) {
      ml_w[wave][0][col] = m[0];
      ml_w[wave][1][col] = l[0];
    }
    __syncthreads();
#pragma unroll 1
    for (int it = threadIdx.x; it < R * (D / 4); it += 256) {
      const int r = it / (D / 4), d = it % (D / 4) * 4, r16 = r & 15, w0 = r >> 4;
      float mr = kKvNone, lr = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < WT; ++w) mr = fmaxf(mr, ml_w[w0 + w * WR][0][r16]);
#pragma unroll
      for (int w = 0; w < WT; ++w) {
        const float f = __builtin_amdgcn_exp2f(ml_w[w0 + w * WR][0][r16] - mr);
        lr = __builtin_fmaf(f, ml_w[w0 + w * WR][1][r16], lr);
        const f4 v = *reinterpret_cast<const f4 *>(&acc_w[w0 + w * WR][r16][d]);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = __builtin_fmaf(f, v[e], x[e]);
      }
      sink.template put<4>(r, mr, lr, d, x);
    }
    if (!whole) sink.join(a.arrivals + part.b * Hkv + h, split, S, is_last);
  }
}

// ---- many rows: the waves own rows and share the keys through LDS ----------------------------------

// A step's codes are converted once per workgroup: a wave reads its share of them from the cache, converts it and writes
// operand registers to LDS (1 KB each, lane by lane, so reads and writes are free of bank conflicts), from where every
// wave feeds its matrix instructions. Two buffers, one barrier a step: a step is written while the one before it is
// used, and its codes were asked for one step earlier still. The pages and scales of 128 blocks of 16 keys at a time
// go through LDS as well (scalar loads would be waited for with every wait for LDS data).
// The last units first: with a causal mask they have the most keys.
template <int D, int NCT, bool TWO>
__global__ void __launch_bounds__(256, NCT > 1 || D == 256 || (TWO && D == 192) ? 2 : TWO || D == 192 ? 3 : 4) k_kv_attn_rows(const KvAttnArgs a) {
  constexpr int C = D / 64, R = 64 * NCT, NQ = TWO ? 2 : 1;
  __shared__ h8 tile[2][8 * C][64];  // K of block n: 2 (n C + c) + y; V: 4 C + 4 c + d, its first four values of block 0
  __shared__ u4 meta[2][128];        // a block's page, K scale, V exponent e and 2^-e
  const int lane = threadIdx.x & 63, col = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int Hkv = a.c.Hkv, h = blockIdx.x % Hkv, S = gridDim.y, split = blockIdx.y;
  const int ps = a.c.ps, in_page = (1 << ps) - 1;
  KvTile t;
  if (!kv_tile_unit(a, R, gridDim.x / Hkv - 1 - blockIdx.x / Hkv, t)) return;
  kv_tile_keys(a, R, t);
  const int t0 = kv_split(t.steps, split, S), t1 = kv_split(t.steps, split + 1, S);
  const int last_page = t.ctx > 0 ? (t.ctx - 1) >> ps : 0;
  const uint32_t koff = col * D + 16 * g4, voff = 4 * (g4 * D + 4 * col);

  // Blocks 128 batch .. of this split. A block behind the sequence's end takes the last page (its keys are masked); one
  // outside the cache reads page 0 with a NaN scale.
  auto ask = [&](int batch) {
    for (int i = threadIdx.x; i < 128; i += 256) {
      const int at = ((t.k0 >> 4) + 2 * t0 + 128 * batch + i) >> (ps - 4);
      const int pg = t.table[at < last_page ? at : last_page];
      const bool bad = static_cast<uint32_t>(pg) >= static_cast<uint32_t>(a.c.n_pages);
      if (bad) kv_flag(a.b.status, kKvBadPage);
      const int64_t ph = static_cast<int64_t>(bad ? 0 : pg) * Hkv + h;
      const int e = bad ? 0 : static_cast<int>((__float_as_uint(a.c.Vs[ph]) >> 23) & 0xffu) - 127;
      meta[batch & 1][i] = u4{static_cast<uint32_t>(bad ? 0 : pg), bad ? 0x7fc00000u : __float_as_uint(a.c.Ks[ph]),
                              __float_as_uint(static_cast<float>(e)), static_cast<uint32_t>(127 - e) << 23};
    }
  };
  auto block_meta = [&](int st, int n) -> const u4 & { return meta[(st - t0) >> 6 & 1][(2 * (st - t0) + n) & 127]; };
  // 64 dims of a block of 16 keys are a unit: the step's 2 C units of K, then 2 C of V, are dealt to the four waves in turn.
  // This wave's unit i: is it K's (known at compile time for all but a mixed turn), which block and dims.
  auto unit = [&](int i) { return wave + 4 * i; };
  auto is_k = [&](int i) { return 4 * (i + 1) <= 2 * C || (4 * i < 2 * C && unit(i) < 2 * C); };
  auto block_of = [&](int i) { return (is_k(i) ? unit(i) : unit(i) - 2 * C) / C; };
  auto dims_of = [&](int i) { return unit(i) % C; };
  u2 coming[C];  // page and K scale of the blocks that are fetched next
  u4 code[C];
  uint32_t ks[C];
  auto peek = [&](int st) {
#pragma unroll
    for (int i = 0; i < C; ++i) coming[i] = *reinterpret_cast<const u2 *>(&block_meta(st, block_of(i)));
  };
  auto fetch = [&](int st) {
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int pg = __builtin_amdgcn_readfirstlane(coming[i].x);
      ks[i] = __builtin_amdgcn_readfirstlane(coming[i].y);
      const int64_t at = (((static_cast<int64_t>(pg) * Hkv + h) << ps) + ((t.k0 + 32 * st + 16 * block_of(i)) & in_page)) * D;
      const uint8_t *base = (is_k(i) ? a.c.K + 64 * dims_of(i) : a.c.V + 256 * dims_of(i)) + at;
      code[i] = *reinterpret_cast<const u4 *>(base + (is_k(i) ? koff : voff));
    }
    peek(st + 1 < t1 ? st + 1 : st);
  };
  auto write = [&](int st) {
    const int buf = st & 1, tok = t.k0 + 32 * st;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      if (is_k(i)) {
        tile[buf][2 * unit(i)][lane] = kv_dec8(code[i].x, code[i].y);
        tile[buf][2 * unit(i) + 1][lane] = kv_dec8(code[i].z, code[i].w);
      } else {
        const int n = block_of(i), c = dims_of(i);
        const bool bad = (ks[i] & 0x7fffffffu) > 0x7f800000u;
        if (tok + 32 > t.ctx || bad) {
          // slots behind the sequence's end were never written: their V codes may be anything, NaN included
          const int left = bad ? 0 : t.ctx - (tok + 16 * n + 4 * g4);
          const uint32_t keep = left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << (8 * left)) - 1;
#pragma unroll
          for (int d = 0; d < 4; ++d) code[i][d] &= keep;
        }
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          h2 x, y;
          kv_dec4(code[i][d], x, y);
          reinterpret_cast<h4 *>(&tile[buf][4 * C + 4 * c + d][lane])[n] = h4{x.x, x.y, y.x, y.y};
        }
      }
    }
  };

  if (t0 < t1) ask(0);
  __syncthreads();
  if (t0 < t1) {
    peek(t0);
    fetch(t0);
  }
  KvRows<C, TWO> q[NCT];
  KvFar far = {kv_move(TWO), 0.f};
  float m[NCT], l[NCT];
  f4 acc[NCT][4 * C];
#pragma unroll
  for (int ct = 0; ct < NCT; ++ct) {
    kv_load_rows<C, TWO>(a, t, t.r0 + (wave * NCT + ct) * 16, h, q[ct]);
    m[ct] = kKvNone;
    l[ct] = t.past ? __builtin_nanf("") : 0.f;
#pragma unroll
    for (int d = 0; d < 4 * C; ++d) acc[ct][d] = f4{0.f, 0.f, 0.f, 0.f};
  }
  if (t0 < t1) {
    write(t0);
    fetch(t0 + 1 < t1 ? t0 + 1 : t0);
  }
  __syncthreads();

  // (The last steps write and fetch as well, the last step again, which nothing reads: a load under a condition would have to
  // be waited for where the two ways meet.)
  for (int st = t0; st < t1; ++st) {
    const int buf = st & 1, tok = t.k0 + 32 * st;
    const u4 m0 = block_meta(st, 0), m1 = block_meta(st, 1);
    h8 kf[2 * C];
#pragma unroll
    for (int c = 0; c < 2 * C; ++c) kf[c] = tile[buf][c][lane];
    write(st + 1);
    if (((st - t0) & 63) == 32 && st - t0 + 32 < t1 - t0) ask(((st - t0) >> 6) + 1);
    fetch(st + 2 < t1 ? st + 2 : t1 - 1);
    f4 s[NCT][2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
      for (int ct = 0; ct < NCT; ++ct) s[ct][n] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 2 * C; ++c)
#pragma unroll
        for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
          for (int z = 0; z < NQ; ++z)
            s[ct][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[c], q[ct].f[c][z], s[ct][n], 0, 0, 0);
      if (n == 0) {
#pragma unroll
        for (int c = 0; c < 2 * C; ++c) kf[c] = tile[buf][2 * C + c][lane];
      }
    }
    const float sk[2] = {__uint_as_float(m0.y), __uint_as_float(m1.y)}, ev[2] = {__uint_as_float(m0.z), __uint_as_float(m1.z)},
                iv[2] = {__uint_as_float(m0.w), __uint_as_float(m1.w)};
    h8 vf[2 * C];
#pragma unroll
    for (int d = 0; d < 2 * C; ++d) vf[d] = tile[buf][4 * C + d][lane];
    h8 p[NCT][NQ];
    kv_weights<NCT, C, TWO>(s, q, sk, ev, iv, tok, tok < t.free0 || tok + 32 > t.free1, far, m, l, acc, p);
#pragma unroll
    for (int d = 0; d < 4 * C; ++d) {
#pragma unroll
      for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
        for (int z = 0; z < NQ; ++z) acc[ct][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[d % (2 * C)], p[ct][z], acc[ct][d], 0, 0, 0);
      if (d < 2 * C) vf[d] = tile[buf][6 * C + d][lane];
    }
    __syncthreads();
  }

  const KvSink<D, R, TWO, false> sink{a, t, h, S == 1, a.part + (static_cast<int64_t>(blockIdx.x) * S + split) * (R * (D + 2))};
  kv_settle<NCT, C, TWO>(far, m, l, acc);
#pragma unroll
  for (int ct = 0; ct < NCT; ++ct) {
    l[ct] = col_sum(l[ct]);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float x[16];  // dims 64 c + 16 g4 + 4 e + d
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * e + d] = acc[ct][4 * c + d][e];
      sink.template put<16>((wave * NCT + ct) * 16 + col, m[ct], l[ct], 64 * c + 16 * g4, x);
    }
  }
}

// The splits' results of k_kv_attn_rows, joined in split order: workgroup (tile and head, 8 rows), each thread four dims at a
// time. In the same launch, as k_kv_attn_keys does it, one workgroup would read all S R (D + 2) floats alone.
template <int D, int R, bool TWO>
__global__ void __launch_bounds__(256) k_kv_attn_join(const KvAttnArgs a, int S) {
  const int Hkv = a.c.Hkv, h = blockIdx.x % Hkv;
  KvTile t;
  if (!kv_tile_unit(a, R, gridDim.x / Hkv - 1 - blockIdx.x / Hkv, t)) return;
  const float *all = a.part + static_cast<int64_t>(blockIdx.x) * S * (R * (D + 2));
  const KvSink<D, R, TWO, false> sink{a, t, h, true, nullptr};
  const int r0 = blockIdx.y * 8, left = t.rows - t.r0 - r0, items = (left < 8 ? left : 8) * (D / 4);
  for (int it = threadIdx.x; it < items; it += 256) sink.template finish_joined<1, 4, false>(all, R * (D + 2), S, r0 * (D / 4) + it, 256, r0 * (D / 4) + items);
}

}  // namespace vybdq
