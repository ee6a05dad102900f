// Attention over the paged 8-bit cache (layout: kv.h), gfx950: from single tokens of many sequences to prompt
// chunks, grouped heads, causal, with or without a sliding window.
//
//   t_ij = (q_i . k_j) scale log2(e) 2^ek + ev     (ek, ev: exponents of key j's page for K and V)
//   w_ij = 2^(t_ij - m_i), acc_i = sum_j w_ij v_j, l_i = sum_j w_ij 2^-ev, o_i = acc_i / l_i
// with v_j, k_j the bare codes: the K scale is one factor per 16 keys in the exponent's fma, and the V scale rides
// in the exponent too, so no code is ever multiplied by its scale. m_i is a running reference that follows the
// largest t: w stays within 2^15, whatever the pages' scales are. One pass over the keys.
//
// Matrix instructions (16x16x32 fp16, float32 sums) on transposed products, so that nothing is ever moved between
// lanes: S^T = K Q^T puts 4 consecutive keys of one query row in a lane, and that is already the layout in which
// O^T = V^T P^T wants P^T, the order of the 32 keys within an instruction being free. K and V codes go from the
// cache straight into operand registers (16-byte loads, one e4m3 -> fp16 conversion per two codes; every e4m3
// value is an fp16 value). Rounded to fp16: the query row, scaled by the power of two that brings its largest
// value into [2^14, 2^15) (exact for fp16 and bf16 values within 2^-38 of the largest), and w (11 bits down to
// 2^-26 of the row's largest). For float32 queries both are split into two fp16 terms (22 bits).
//
// A wave owns 16 NCT query rows (row = token * G + head of the group; the G query heads of a key head read the
// same keys, so they share its tiles). WT waves of a workgroup take turns over the keys (32 at a time) and are
// joined through LDS; WR waves own different rows. With few rows the keys are split over workgroups too (gridDim.y):
// each stores its (m, l, acc), and the last one to arrive joins them in split order, so results do not depend
// on the order of arrival.
#pragma once

#include "kv.h"

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
  int32_t per_seq;     // 1: a workgroup takes every tile of one sequence; 0: one tile
  float scale2;        // scale * log2(e)
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

// 16 consecutive elements of a row as float32
__device__ __forceinline__ void load16(const void *p, int dt, int64_t i, float (&x)[16]) {
  if (dt == VYBDQ_F32) {
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
        if (dt == VYBDQ_F16) {
          x[8 * j + 2 * e] = half_bits_to_f32(w & 0xffffu);
          x[8 * j + 2 * e + 1] = half_bits_to_f32(w >> 16);
        } else {
          x[8 * j + 2 * e] = __uint_as_float(w << 16);
          x[8 * j + 2 * e + 1] = __uint_as_float(w & 0xffff0000u);
        }
      }
    }
  }
}

// N consecutive outputs (N a multiple of 4), rounded once to the output type
template <int N>
__device__ __forceinline__ void store_n(void *p, int dt, int64_t i, const float (&x)[N]) {
  if (dt == VYBDQ_F32) {
    f4 *o = reinterpret_cast<f4 *>(static_cast<float *>(p) + i);
#pragma unroll
    for (int j = 0; j < N / 4; ++j) o[j] = f4{x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]};
  } else {
    u2 *o = reinterpret_cast<u2 *>(static_cast<uint16_t *>(p) + i);
#pragma unroll
    for (int j = 0; j < N / 4; ++j) {
      uint16_t r[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        r[e] = dt == VYBDQ_F16 ? __builtin_bit_cast(uint16_t, static_cast<_Float16>(x[4 * j + e]))
                               : f32_to_bf16(x[4 * j + e]);
      o[j] = u2{r[0] | (static_cast<uint32_t>(r[1]) << 16), r[2] | (static_cast<uint32_t>(r[3]) << 16)};
    }
  }
}

constexpr float kKvRef = 12.0f;   // a row's reference is 2^-12 of its largest weight when it is taken
constexpr float kKvMove = 15.0f;  // and is taken anew once a weight would pass 2^15
#define KV_NEG_INF (-__builtin_inff())

// LDS floats a workgroup joins its WT waves through: one column tile at a time
template <int D, int WT>
constexpr int kv_join_floats() {
  return WT > 1 ? WT * 16 * (D + 4 + 2) : 1;
}

template <int D, int NCT, int WT, int WR, bool SPLIT2>
__global__ void __launch_bounds__(64 * WT * WR) k_kv_attn(const KvAttnArgs a) {
  constexpr int C = D / 64, R = 16 * NCT * WR, NW = WT * WR, NQ = SPLIT2 ? 2 : 1;
  __shared__ float join[kv_join_floats<D, WT>()];
  __shared__ bool is_last;
  const int lane = threadIdx.x & 63, col = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wt = WT > 1 ? wave % WT : 0, wr = WR > 1 ? wave / WT : 0;
  const int Hkv = a.c.Hkv, h = blockIdx.x % Hkv, S = gridDim.y, split = blockIdx.y;
  const int unit = blockIdx.x / Hkv, G = a.G, ps = a.c.ps, P = 1 << ps;
  int b = unit;
  int64_t tile = 0;
  if (!a.per_seq) {
    // sequence b's tiles are units first(b) ..: ceil(n G / R) of them, and floor((s + n) G / R) - floor(s G / R) + 1
    // is no less. The last units first: with a causal mask they have the most keys.
    const int64_t u = static_cast<int64_t>(gridDim.x / Hkv) - 1 - unit;
    auto first = [&](int i) { return static_cast<int64_t>(a.b.q_start[i]) * G / R + i; };
    b = kv_find(a.b.B, u, first);
    tile = u - first(b);
    if (tile < 0) return;
  }
  const KvSeq sq = kv_seq(a.b, b);
  const int64_t rows = static_cast<int64_t>(sq.n) * G;
  if (rows == 0) return;
  // tokens past the table's pages: the sequence's rows are NaN
  const bool past = sq.ctx > (a.b.W << ps);
  if (past && (threadIdx.x & 63) == 0) kv_flag(a.b.status, kKvBadCtx);
  const int ctx = sq.ctx > 0 && !past ? sq.ctx : 0, p0 = ctx - sq.n;
  const int32_t *table = a.b.table + static_cast<int64_t>(b) * a.b.W;

  for (int64_t r0 = tile * R; r0 < rows; r0 += R) {
    // a tile beyond the first that the launch did not plan for is not split: split 0 takes all its keys
    const bool whole = S == 1 || (a.per_seq && r0 > 0);
    if (whole && split > 0) return;
    // keys that some row of the tile sees: [k0, k1), in steps of 32
    const int i_lo = static_cast<int>(r0 / G);
    const int i_hi = static_cast<int>((r0 + R < rows ? r0 + R : rows) - 1) / G;
    int k1 = a.causal ? p0 + i_hi + 1 : ctx;
    k1 = k1 > 0 ? k1 : 0;
    int k0 = a.window ? p0 + i_lo - a.window + 1 : 0;
    k0 = (k0 > 0 ? k0 : 0) & ~31;
    const int steps = k1 > k0 ? (k1 - k0 + 31) >> 5 : 0;
    const int t0 = whole ? 0 : static_cast<int>(static_cast<int64_t>(steps) * split / S);
    const int t1 = whole ? steps : static_cast<int>(static_cast<int64_t>(steps) * (split + 1) / S);
    // keys that every row sees need no mask
    const int free0 = a.window ? p0 + i_hi - a.window + 1 : 0, free1 = a.causal ? p0 + i_lo + 1 : ctx;

    // this lane's query rows
    h8 qf[NCT][2 * C][NQ];
    float qc[NCT], m[NCT], l[NCT];
    int lo_r[NCT], hi_r[NCT];
    f4 acc[NCT][4 * C];
#pragma unroll
    for (int ct = 0; ct < NCT; ++ct) {
      const int64_t r = r0 + (wr * NCT + ct) * 16 + col;
      const bool have = r < rows;
      const int64_t rr = have ? r : 0;
      const int i = static_cast<int>(rr / G), hq = h * G + static_cast<int>(rr % G);
      hi_r[ct] = !have ? 0 : a.causal ? p0 + i + 1 : ctx;
      lo_r[ct] = a.window ? p0 + i - a.window + 1 : 0;
      const int64_t at = (sq.s0 + i) * a.ldq + static_cast<int64_t>(hq) * D + 16 * g4;
      float amax = 0.f;
      bool bad = false;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float x[16];
        load16(a.q, a.dt, at + 64 * c, x);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          bad |= (__float_as_uint(x[e]) & 0x7fffffffu) >= 0x7f800000u;
          amax = fmaxf(amax, fabsf(x[e]));
        }
      }
      float inv;
      const float sc = block_scale(col_max(amax), inv);
      // an infinity or NaN in any of the row's four lanes makes its scores NaN
      qc[ct] = sc * a.scale2 + col_sum(bad ? __builtin_nanf("") : 0.f);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float x[16];
        load16(a.q, a.dt, at + 64 * c, x);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float v = x[e] * inv;
          const _Float16 f = static_cast<_Float16>(v);
          qf[ct][2 * c + e / 8][0][e % 8] = f;
          if constexpr (SPLIT2) qf[ct][2 * c + e / 8][NQ - 1][e % 8] = static_cast<_Float16>(v - static_cast<float>(f));
        }
      }
      m[ct] = KV_NEG_INF;
      l[ct] = past ? __builtin_nanf("") : 0.f;
#pragma unroll
      for (int t = 0; t < 4 * C; ++t) acc[ct][t] = f4{0.f, 0.f, 0.f, 0.f};
    }

    for (int st = t0 + wt; st < t1; st += WT) {
      const int tok = k0 + 32 * st;
      // the two blocks of 16 keys: where they lie, and their scales
      const uint8_t *kb[2], *vb[2];
      float ks[2], ev[2], iv[2];
      bool drop[2];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const int t = tok + 16 * n, at = t >> ps;
        const bool in = t < ctx;
        const int pg = in ? table[at] : 0;
        drop[n] = pg < 0 || pg >= a.c.n_pages;
        const int64_t ph = static_cast<int64_t>(drop[n] ? 0 : pg) * Hkv + h;
        const int64_t off = ((ph << ps) + (t & (P - 1))) * D;
        kb[n] = a.c.K + off;
        vb[n] = a.c.V + off;
        const uint32_t e = in && !drop[n] ? (__float_as_uint(a.c.Vs[ph]) >> 23) & 0xffu : 127u;
        ks[n] = drop[n] ? __builtin_nanf("") : in ? a.c.Ks[ph] : 1.0f;
        ev[n] = static_cast<float>(static_cast<int>(e) - 127);
        iv[n] = __uint_as_float((254u - e) << 23);
        if (drop[n] && lane == 0) kv_flag(a.b.status, kKvBadPage);
      }
      u4 kw[2][C], vw[2][C];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int c = 0; c < C; ++c) {
          kw[n][c] = *reinterpret_cast<const u4 *>(kb[n] + col * D + 64 * c + 16 * g4);
          vw[n][c] = *reinterpret_cast<const u4 *>(vb[n] + 4 * (g4 * D + 64 * c + 4 * col));
        }
      f4 s[NCT][2];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
#pragma unroll
        for (int ct = 0; ct < NCT; ++ct) s[ct][n] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const h8 kf = kv_dec8(kw[n][c][2 * x], kw[n][c][2 * x + 1]);
#pragma unroll
            for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
              for (int y = 0; y < NQ; ++y)
                s[ct][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[ct][2 * c + x][y], s[ct][n], 0, 0, 0);
          }
      }
      // slots behind the sequence's end were never written: their V codes may be anything, NaN included
      if (tok + 32 > ctx || drop[0] || drop[1]) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const int left = drop[n] ? 0 : ctx - (tok + 16 * n + 4 * g4);
          const uint32_t keep = left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << (8 * left)) - 1;
#pragma unroll
          for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) vw[n][c][e] &= keep;
        }
      }
      const bool masked = tok < free0 || tok + 32 > free1;
      h8 pf[NCT][NQ];
#pragma unroll
      for (int ct = 0; ct < NCT; ++ct) {
        float t[8];
        float top = KV_NEG_INF;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float ck = qc[ct] * ks[n];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            t[4 * n + e] = __builtin_fmaf(s[ct][n][e], ck, ev[n]);
            if (masked) {
              const int key = tok + 16 * n + 4 * g4 + e;
              t[4 * n + e] = key >= lo_r[ct] && key < hi_r[ct] ? t[4 * n + e] : KV_NEG_INF;
            }
            top = fmaxf(top, t[4 * n + e]);
          }
        }
        if (__ballot(top > m[ct] + kKvMove)) {
          const float now = fmaxf(m[ct], col_max(top) - kKvRef);
          const float f = now == KV_NEG_INF ? 1.0f : __builtin_amdgcn_exp2f(m[ct] - now);
          m[ct] = now;
          l[ct] *= f;
#pragma unroll
          for (int d = 0; d < 4 * C; ++d) acc[ct][d] *= f;
        }
        const float ref = m[ct] == KV_NEG_INF ? 0.f : m[ct];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float w = __builtin_amdgcn_exp2f(t[4 * n + e] - ref);
            l[ct] = __builtin_fmaf(w, iv[n], l[ct]);
            const _Float16 f = static_cast<_Float16>(w);
            pf[ct][0][4 * n + e] = f;
            if constexpr (SPLIT2) pf[ct][NQ - 1][4 * n + e] = static_cast<_Float16>(w - static_cast<float>(f));
          }
      }
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const h8 vf = kv_dec8(vw[0][c][d], vw[1][c][d]);
#pragma unroll
          for (int ct = 0; ct < NCT; ++ct)
#pragma unroll
            for (int y = 0; y < NQ; ++y)
              acc[ct][4 * c + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[ct][y], acc[ct][4 * c + d], 0, 0, 0);
        }
    }

    // ---- the tile's rows: joined over the waves, then stored, or left for the last split
    float *part = a.part + (static_cast<int64_t>(blockIdx.x) * S + split) * (R * (D + 2));
    auto put = [&](int r, float mr, float lr, int d, const auto &x) {  // dims d .. of tile row r
      constexpr int N = sizeof(x) / 4;
      if (whole) {
        const int64_t rr = r0 + r;
        if (rr >= rows) return;
        const int64_t at = (sq.s0 + rr / G) * (static_cast<int64_t>(Hkv) * G) + h * G + rr % G;
        const float f = lr == 0.f ? 0.f : 1.0f / lr;
        float y[N];
#pragma unroll
        for (int e = 0; e < N; ++e) y[e] = x[e] * f;
        store_n<N>(a.out, a.dt, at * D + d, y);
        if (a.lse && d == 0) a.lse[at] = lr == 0.f ? KV_NEG_INF : (mr + __builtin_amdgcn_logf(lr)) * 0.6931471805599453f;
      } else if (r0 + r < rows) {
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
    };
#pragma unroll
    for (int ct = 0; ct < NCT; ++ct) {
      l[ct] = col_sum(l[ct]);
      if constexpr (WT == 1) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
          float x[16];  // dims 64 c + 16 g4 + 4 e + d
#pragma unroll
          for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * e + d] = acc[ct][4 * c + d][e];
          put((wr * NCT + ct) * 16 + col, m[ct], l[ct], 64 * c + 16 * g4, x);
        }
      } else {
        float *acc_w = join + wave * (16 * (D + 4)), *m_w = join + WT * 16 * (D + 4), *l_w = m_w + WT * 16;
        if (ct > 0 || r0 > tile * R) __syncthreads();
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            *reinterpret_cast<f4 *>(acc_w + col * (D + 4) + 64 * c + 16 * g4 + 4 * e) =
                f4{acc[ct][4 * c][e], acc[ct][4 * c + 1][e], acc[ct][4 * c + 2][e], acc[ct][4 * c + 3][e]};
        if (g4 == 0) {
          m_w[wt * 16 + col] = m[ct];
          l_w[wt * 16 + col] = l[ct];
        }
        __syncthreads();
        for (int it = threadIdx.x; it < 16 * (D / 4); it += 64 * NW) {
          const int r = it / (D / 4), d = it % (D / 4) * 4;
          float mr = KV_NEG_INF, lr = 0.f;
#pragma unroll
          for (int w = 0; w < WT; ++w) mr = fmaxf(mr, m_w[w * 16 + r]);
          const float ref = mr == KV_NEG_INF ? 0.f : mr;
          float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int w = 0; w < WT; ++w) {
            const float f = __builtin_amdgcn_exp2f(m_w[w * 16 + r] - ref);
            lr = __builtin_fmaf(f, l_w[w * 16 + r], lr);
            const f4 v = *reinterpret_cast<const f4 *>(join + w * (16 * (D + 4)) + r * (D + 4) + d);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = __builtin_fmaf(f, v[e], x[e]);
          }
          put(ct * 16 + r, mr, lr, d, x);
        }
      }
    }
    if (!whole) {
      // arrival: the partials are stored through the XCD's L2 and have completed before it is counted; the last
      // one resets the counter and reads the others' with device-coherent loads
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (threadIdx.x == 0) {
        const uint32_t old = __hip_atomic_fetch_add(a.arrivals + blockIdx.x, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        is_last = old == static_cast<uint32_t>(S - 1);
        if (is_last) __hip_atomic_store(a.arrivals + blockIdx.x, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
      __syncthreads();
      if (is_last) {
        const float *all = a.part + static_cast<int64_t>(blockIdx.x) * S * (R * (D + 2));
        const int n_rows = rows - r0 < R ? static_cast<int>(rows - r0) : R;
        for (int it = threadIdx.x; it < n_rows * (D / 2); it += 64 * NW) {
          const int r = it / (D / 2), d = it % (D / 2) * 2;
          float mr = KV_NEG_INF, lr = 0.f, x0 = 0.f, x1 = 0.f;
          for (int w0 = 0; w0 < S; w0 += 8) {
            uint64_t ml[8], v[8];
#pragma unroll
            for (int w = 0; w < 8; ++w)
              if (w0 + w < S) {
                const float *pw = all + static_cast<int64_t>(w0 + w) * (R * (D + 2));
                ml[w] = __hip_atomic_load(reinterpret_cast<const uint64_t *>(pw) + r, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                v[w] = __hip_atomic_load(reinterpret_cast<const uint64_t *>(pw + 2 * R + r * D + d), __ATOMIC_RELAXED,
                                         __HIP_MEMORY_SCOPE_AGENT);
              }
            float now = mr;
#pragma unroll
            for (int w = 0; w < 8; ++w)
              if (w0 + w < S) now = fmaxf(now, __uint_as_float(static_cast<uint32_t>(ml[w])));
            const float ref = now == KV_NEG_INF ? 0.f : now;
            const float f0 = __builtin_amdgcn_exp2f(mr - ref);
            lr *= f0;
            x0 *= f0;
            x1 *= f0;
            mr = now;
#pragma unroll
            for (int w = 0; w < 8; ++w)
              if (w0 + w < S) {
                const float f = __builtin_amdgcn_exp2f(__uint_as_float(static_cast<uint32_t>(ml[w])) - ref);
                lr = __builtin_fmaf(f, __uint_as_float(static_cast<uint32_t>(ml[w] >> 32)), lr);
                x0 = __builtin_fmaf(f, __uint_as_float(static_cast<uint32_t>(v[w])), x0);
                x1 = __builtin_fmaf(f, __uint_as_float(static_cast<uint32_t>(v[w] >> 32)), x1);
              }
          }
          const int64_t rr = r0 + r;
          const int64_t at = (sq.s0 + rr / G) * (static_cast<int64_t>(Hkv) * G) + h * G + rr % G;
          const float f = lr == 0.f ? 0.f : 1.0f / lr;
          if (a.dt == VYBDQ_F32) *reinterpret_cast<f2 *>(static_cast<float *>(a.out) + at * D + d) = f2{x0 * f, x1 * f};
          else {
            const uint16_t u = a.dt == VYBDQ_F16 ? __builtin_bit_cast(uint16_t, static_cast<_Float16>(x0 * f)) : f32_to_bf16(x0 * f);
            const uint16_t v = a.dt == VYBDQ_F16 ? __builtin_bit_cast(uint16_t, static_cast<_Float16>(x1 * f)) : f32_to_bf16(x1 * f);
            *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(a.out) + at * D + d) = u | (static_cast<uint32_t>(v) << 16);
          }
          if (a.lse && d == 0) a.lse[at] = lr == 0.f ? KV_NEG_INF : (mr + __builtin_amdgcn_logf(lr)) * 0.6931471805599453f;
        }
      }
    }
    if (!a.per_seq) break;
  }
}

}  // namespace vybdq
