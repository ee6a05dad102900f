// Appending keys and values to the paged 8-bit cache (layout: kv.h), with the position rotation of q and k on
// the way, gfx950.
//
//   y_a = x_a c - x_b s, y_b = x_b c + x_a s   for the pairs (a, b) of the first R dims: (i, i + R / 2), or
//     (2 i, 2 i + 1) interleaved; c, s = cos, sin [position][i], float32. Contraction is off: every product and
//     sum rounds once to float32, so codes do not depend on how a compiler fuses them.
//   e = the least integer with amax <= 448 * 2^e over a page's new tokens of one head (k rotated), in
//     [-60, 60]; where the page keeps earlier tokens, at least its old e. scale = 2^e, code = e4m3(y * 2^-e),
//     ties to even. If e grows, the kept codes become e4m3(code * 2^(e_old - e)): a change of exponent, exact but
//     for values that fall among e4m3's subnormals (below 2^-15 of the page's largest), which is why the scale
//     is a power of two.
// A token of which a rotated k or a v of a head is an infinity or NaN gets codes that no finite token has there:
// k NaN, v zero. Its score is then NaN for the rows that see it, and a row that does not see it multiplies zeros.
//
// One workgroup per (page that a sequence's rows reach, key/value head): it alone writes that page's codes and scales.
// A thread reads 16 dims of a token's k (both halves of its pairs) and 4 dims of four slots of v and keeps them in registers
// until the page's largest magnitude is known (512 threads: all of a page of 64 tokens of 128 dims); of a larger page the
// rest is read again (from L2). Query heads are rotated by workgroups of their own (gridDim.y), which need not wait for a page's
// magnitude; a thread rotates up to four heads of its group by the angles that it has read (one head each: 39.9 us
// against 36.5 below).
//
// Bound by memory when there is much of it, MI355X: five prompts of up to 1638 tokens, 32 / 8 heads of 128, bf16, 127 MB:
// 36.5 us, 3.5 TB/s; seven of up to 301 tokens, 24 / 4 heads of 256, float32, 85 MB: 20.9 us, 4.1 TB/s (a large copy runs
// at 4.7). A decode step takes 6 us on the GPU for one sequence and 7 for 128, about 2 of them the launch; asking for k and v
// before the page is known, or for the old codes of a group of slots before the page's magnitude is, changed neither.
#include "kv.h"

#include <mutex>
#include <string>

namespace vybdq {

static __device__ __align__(256) uint32_t kv_status_word[64] = {0};

namespace {
std::mutex g_kv_mu;
uint32_t *g_kv_status[64];
}  // namespace

// the current device's status word (hipGetSymbolAddress once per device)
int kv_status_address(uint32_t *&ptr) {
  int dev = -1;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64)
    return set_error(VYBDQ_ERR_HIP, "vybdq_kv: no current HIP device");
  std::lock_guard<std::mutex> lock(g_kv_mu);
  if (!g_kv_status[dev]) {
    void *p = nullptr;
    const hipError_t e = hipGetSymbolAddress(&p, HIP_SYMBOL(kv_status_word));
    if (e != hipSuccess || !p)
      return set_error(VYBDQ_ERR_HIP, std::string("vybdq_kv: hipGetSymbolAddress failed: ") + hipGetErrorString(e));
    g_kv_status[dev] = static_cast<uint32_t *>(p);
  }
  ptr = g_kv_status[dev];
  return VYBDQ_OK;
}

// What was reported so far, taken and cleared in one step: a call that another thread has launched meanwhile may report more.
__global__ void k_kv_status_take(uint32_t *status) {
  status[1] = __hip_atomic_exchange(status, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

struct KvAppendArgs {
  KvCacheArgs c;
  KvBatchArgs b;
  const void *k, *v, *q;
  void *q_out;
  const float *cosv, *sinv;
  int64_t ldk, ldv, ldq;
  int32_t G, R, n_pos, inter;
  int32_t per_seq;  // 1: workgroup (b, head) takes every page of sequence b; 0: one page per workgroup
};

// 8 elements as they lie in memory, and as float32
template <int DT>
struct KvEight {
  u4 w[DT == VYBDQ_F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void *p, int64_t i) {
    const u4 *s = reinterpret_cast<const u4 *>(static_cast<const uint8_t *>(p) + i * (DT == VYBDQ_F32 ? 4 : 2));
    w[0] = s[0];
    if constexpr (DT == VYBDQ_F32) w[1] = s[1];
  }
  __device__ __forceinline__ void unpack(float (&x)[8]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (DT == VYBDQ_F32) {
        x[j] = __uint_as_float(w[0][j]);
        x[4 + j] = __uint_as_float(w[1][j]);
      } else if constexpr (DT == VYBDQ_F16) {
        x[2 * j] = half_bits_to_f32(w[0][j] & 0xffffu);
        x[2 * j + 1] = half_bits_to_f32(w[0][j] >> 16);
      } else {
        x[2 * j] = __uint_as_float(w[0][j] << 16);
        x[2 * j + 1] = __uint_as_float(w[0][j] & 0xffff0000u);
      }
    }
  }
};

template <int DT>
__device__ __forceinline__ void load_n(const void *p, int64_t i, float (&x)[8]) {
  KvEight<DT> r;
  r.load(p, i);
  r.unpack(x);
}

template <int DT>
__device__ __forceinline__ void load_n(const void *p, int64_t i, float (&x)[4]) {
  if constexpr (DT == VYBDQ_F32) {
    const f4 a = *reinterpret_cast<const f4 *>(static_cast<const float *>(p) + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = a[j];
  } else if constexpr (DT == VYBDQ_F16) {
    const h4 a = *reinterpret_cast<const h4 *>(static_cast<const _Float16 *>(p) + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = static_cast<float>(a[j]);
  } else {
    const u2 a = *reinterpret_cast<const u2 *>(static_cast<const uint16_t *>(p) + i);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t w = a[j];
      x[2 * j] = __uint_as_float(w << 16);
      x[2 * j + 1] = __uint_as_float(w & 0xffff0000u);
    }
  }
}

// query heads that a thread rotates by the same angles at most: 64 bytes of cos and sin go with 32 of a bf16 head's piece (of a
// float32 head's 64: two heads 20.8 us where four take 23.3)
constexpr int kv_turn_heads(int dt) { return dt == VYBDQ_F32 ? 2 : 4; }

// Piece i of a row's D / 16: 16 dims that hold both members of their pairs, 8 from dim lo and 8 from dim hi.
struct KvPiece {
  int lo, hi;
};
__device__ __forceinline__ KvPiece kv_piece(const KvAppendArgs &a, int i) {
  const int half = a.R >> 1;
  if (!a.inter && 8 * i < half) return {8 * i, half + 8 * i};
  return {16 * i, 16 * i + 8};  // (pairs of neighbours, or dims behind R)
}

// cos and sin of piece i's pairs at position pos.
__device__ __forceinline__ void kv_turn(const KvAppendArgs &a, int i, int pos, float (&c)[8], float (&s)[8]) {
  const int64_t row = 16 * i < a.R ? static_cast<int64_t>(pos) * (a.R >> 1) + 8 * i : 0;
  if (a.R == 0) return;
  load_n<VYBDQ_F32>(a.cosv, row, c);
  load_n<VYBDQ_F32>(a.sinv, row, s);
}

// Piece i of a row, rotated.
__device__ __forceinline__ void rotate16(const KvAppendArgs &a, int i, const float (&c)[8], const float (&s)[8], float (&x)[2][8]) {
#pragma clang fp contract(off)
  if (16 * i >= a.R) return;
  // (by selects: two branches would be merged into one that indexes x by a variable, in scratch memory)
  float u[8], v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float p = a.inter ? x[j >> 2][2 * (j & 3)] : x[0][j], q = a.inter ? x[j >> 2][2 * (j & 3) + 1] : x[1][j];
    const float pc = p * c[j], qs = q * s[j], qc = q * c[j], ps = p * s[j];
    u[j] = pc - qs;
    v[j] = qc + ps;
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) x[e >> 3][e & 7] = a.inter ? (e & 1 ? v[e >> 1] : u[e >> 1]) : e < 8 ? u[e & 7] : v[e & 7];
}

template <int DT>
__device__ __forceinline__ void store8(void *p, int64_t i, const float (&x)[8]) {
  if constexpr (DT == VYBDQ_F32) {
    f4 *o = reinterpret_cast<f4 *>(static_cast<float *>(p) + i);
    o[0] = f4{x[0], x[1], x[2], x[3]};
    o[1] = f4{x[4], x[5], x[6], x[7]};
  } else if constexpr (DT == VYBDQ_F16) {
    h8 o;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = static_cast<_Float16>(x[j]);
    *reinterpret_cast<h8 *>(static_cast<_Float16 *>(p) + i) = o;
  } else {
    u4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      o[j] = f32_to_bf16(x[2 * j]) | (static_cast<uint32_t>(f32_to_bf16(x[2 * j + 1])) << 16);
    *reinterpret_cast<u4 *>(static_cast<uint16_t *>(p) + i) = o;
  }
}

// Four values times a power of two as e4m3 codes, rounded to nearest even and held to +-448.
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, float inv) {
  auto cl = [&](float x) { return __builtin_amdgcn_fmed3f(x * inv, -kKvCodeMax, kKvCodeMax); };
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(cl(a), cl(b), 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(cl(c), cl(d), lo, true);
}

// Four codes brought to a larger scale (f = 2^(e_old - e)). A NaN code stays one.
__device__ __forceinline__ uint32_t recode4(uint32_t w, float f) {
  const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  const int a = __builtin_amdgcn_cvt_pk_fp8_f32(lo.x * f, lo.y * f, 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(hi.x * f, hi.y * f, a, true);
}

// The least e with amax <= 448 * 2^e (448 = 1.75 * 2^8), within the allowed exponents; a zero has the smallest.
__device__ __forceinline__ int page_exp(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int x = static_cast<int>(u >> 23) - 127;
  const int e = (u & 0x7fffffu) <= 0x600000u ? x - 8 : x - 7;
  return e < kKvExpMin ? kKvExpMin : (e > kKvExpMax ? kKvExpMax : e);
}

__device__ __forceinline__ float exp2i(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v = fmaxf(v, __shfl_xor(v, m));
  return v;
}

// |x| where x is finite, else 0 and `bad`
__device__ __forceinline__ float magnitude(float x, bool &bad) {
  const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
  if (u < 0x7f800000u) return __uint_as_float(u);
  bad = true;
  return 0.0f;
}

template <int DT, int D>
__global__ void __launch_bounds__(512, 4) k_kv_append(const KvAppendArgs a) {
  __shared__ float red[2][8];
  __shared__ int bad_token[256];  // by the token's place among the page's new ones
  constexpr int D16 = D / 16, D4 = D / 4;
  const int tid = threadIdx.x, nthr = blockDim.x, P = 1 << a.c.ps;
  const int Hkv = a.c.Hkv, h = blockIdx.x % Hkv;
  const int u = blockIdx.x / Hkv;
  int b = u;
  int64_t j = 0;
  if (!a.per_seq) {
    // sequence b's pages are units first(b) ..: n rows reach at most ceil(n / P) + 1 pages, and
    // floor((s + n) / P) - floor(s / P) + 2 is no less
    auto first = [&](int i) { return (static_cast<int64_t>(a.b.q_start[i]) >> a.c.ps) + 2 * static_cast<int64_t>(i); };
    b = kv_find(a.b.B, u, first);
    j = u - first(b);
  }
  const KvSeq sq = kv_seq(a.b, b);
  if (!sq.ok || sq.n == 0 || j < 0) return;
  if (sq.ctx < sq.n || (static_cast<int64_t>(sq.ctx) + P - 1) >> a.c.ps > a.b.W) {
    if (tid == 0) kv_flag(a.b.status, kKvBadCtx);
    return;
  }
  if (a.R && sq.ctx > a.n_pos) {
    if (tid == 0) kv_flag(a.b.status, kKvBadAngle);
    return;
  }
  const int p0 = sq.ctx - sq.n;  // position of the first row
  const int last = (sq.ctx - 1) >> a.c.ps;
  if (blockIdx.y > 0) {  // query heads
    for (int64_t i = (p0 >> a.c.ps) + j; i <= last; ++i) {
      const int base = static_cast<int>(i) << a.c.ps, lo = p0 > base ? p0 : base;
      const int nt = (sq.ctx - base < P ? sq.ctx - base : P) - (lo - base);
      const int64_t row0 = sq.s0 + (lo - p0);
      constexpr int kHeads = kv_turn_heads(DT);
      const int chunks = (a.G + kHeads - 1) / kHeads, heads = (a.G + chunks - 1) / chunks, per_token = chunks * D16;
      for (int it = (blockIdx.y - 1) * nthr + tid; it < nt * per_token; it += (gridDim.y - 1) * nthr) {
        const int t = it / per_token, r = it % per_token, d = r % D16, g0 = r / D16 * heads;
        const KvPiece p = kv_piece(a, d);
        const int64_t from = (row0 + t) * a.ldq + (h * a.G + g0) * D, to = ((row0 + t) * Hkv * a.G + h * a.G + g0) * D;
        float c[8], s[8];
        kv_turn(a, d, lo + t, c, s);
        KvEight<DT> raw[kHeads][2];
#pragma unroll
        for (int g = 0; g < kHeads; ++g) {
          const int64_t at = from + (g < heads && g0 + g < a.G ? g : 0) * D;
          raw[g][0].load(a.q, at + p.lo);
          raw[g][1].load(a.q, at + p.hi);
        }
#pragma unroll
        for (int g = 0; g < kHeads; ++g) {
          if (g < heads && g0 + g < a.G) {
            float x[2][8];
            raw[g][0].unpack(x[0]);
            raw[g][1].unpack(x[1]);
            rotate16(a, d, c, s, x);
            store8<DT>(a.q_out, to + g * D + p.lo, x[0]);
            store8<DT>(a.q_out, to + g * D + p.hi, x[1]);
          }
        }
      }
      if (!a.per_seq) break;
    }
    return;
  }
  for (int64_t i = (p0 >> a.c.ps) + j; i <= last; ++i) {
    const int base = static_cast<int>(i) << a.c.ps;
    const int lo = p0 > base ? p0 : base, hi = sq.ctx < base + P ? sq.ctx : base + P;
    const int keep = lo - base, nt = hi - lo;
    const int64_t row0 = sq.s0 + (lo - p0);

    const int pg = a.b.table[static_cast<int64_t>(b) * a.b.W + i];
    const bool valid = pg >= 0 && pg < a.c.n_pages;
    if (!valid && tid == 0) kv_flag(a.b.status, kKvBadPage);
    if (valid) {
      const int64_t ph = static_cast<int64_t>(pg) * Hkv + h;
      uint8_t *Kp = a.c.K + ph * P * D, *Vp = a.c.V + ph * P * D;
      // the old exponents, read before any thread writes the new ones
      auto old_exp = [&](const float *s) {
        const int e = keep ? static_cast<int>((__float_as_uint(s[ph]) >> 23) & 0xffu) - 127 : kKvExpMin;
        return e > kKvExpMax ? kKvExpMax : (e < kKvExpMin ? kKvExpMin : e);
      };
      const int eko = old_exp(a.c.Ks), evo = old_exp(a.c.Vs);
      for (int t = tid; t < nt; t += nthr) bad_token[t] = 0;
      __syncthreads();
      // 1. the largest finite magnitude of the new tokens, and the tokens that hold something else
      const int nk = nt * D16, g0 = keep >> 2, nv = (((keep + nt + 3) >> 2) - g0) * D4;
      auto load_k = [&](int it, float (&x)[2][8]) {
        const int t = it / D16;
        const KvPiece p = kv_piece(a, it % D16);
        const int64_t at = (row0 + t) * a.ldk + h * D;
        load_n<DT>(a.k, at + p.lo, x[0]);
        load_n<DT>(a.k, at + p.hi, x[1]);
        if (16 * (it % D16) >= a.R) return;
        float c[8], s[8];
        kv_turn(a, it % D16, lo + t, c, s);
        rotate16(a, it % D16, c, s, x);
      };
      auto load_v = [&](int it, float (&x)[4][4]) {  // slots 4 g .., dims d ..; slots that are not new: zero
        const int t0 = 4 * (g0 + it / D4) - keep, d = it % D4 * 4;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int t = t0 + r;
#pragma unroll
          for (int e = 0; e < 4; ++e) x[r][e] = 0.f;
          if (t >= 0 && t < nt) load_n<DT>(a.v, (row0 + t) * a.ldv + h * D + d, x[r]);
        }
      };
      float kx[2][8], vx[4][4], mk = 0.f, mv = 0.f;  // this thread's first pieces, held until their codes are known
      auto see_k = [&](int it, const float (&x)[2][8]) {
        bool bad = false;
#pragma unroll
        for (int e = 0; e < 16; ++e) mk = fmaxf(mk, magnitude(x[e >> 3][e & 7], bad));
        if (bad) bad_token[it / D16] = 1;
      };
      auto see_v = [&](int it, const float (&x)[4][4]) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          bool bad = false;
#pragma unroll
          for (int e = 0; e < 4; ++e) mv = fmaxf(mv, magnitude(x[r][e], bad));
          if (bad) bad_token[4 * (g0 + it / D4) - keep + r] = 1;
        }
      };
      if (tid < nk) load_k(tid, kx);
      if (tid < nv) load_v(tid, vx);
      if (tid < nk) see_k(tid, kx);
      if (tid < nv) see_v(tid, vx);
      for (int it = tid + nthr; it < nk; it += nthr) {
        float x[2][8];
        load_k(it, x);
        see_k(it, x);
      }
      for (int it = tid + nthr; it < nv; it += nthr) {
        float x[4][4];
        load_v(it, x);
        see_v(it, x);
      }
      mk = wave_max(mk);
      mv = wave_max(mv);
      if ((tid & 63) == 0) {
        red[0][tid >> 6] = mk;
        red[1][tid >> 6] = mv;
      }
      __syncthreads();
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        mk = fmaxf(mk, w < nthr >> 6 ? red[0][w] : 0.f);
        mv = fmaxf(mv, w < nthr >> 6 ? red[1][w] : 0.f);
      }
      const int ekn = page_exp(mk), evn = page_exp(mv), ek = ekn > eko ? ekn : eko, ev = evn > evo ? evn : evo;
      if (tid == 0) {
        a.c.Ks[ph] = exp2i(ek);
        a.c.Vs[ph] = exp2i(ev);
      }
      const float ik = exp2i(-ek), iv = exp2i(-ev);

      // 2. codes of the new tokens
      auto put_k = [&](int it, const float (&x)[2][8]) {
        const int t = it / D16;
        const KvPiece d = kv_piece(a, it % D16);
        const bool bad = bad_token[t];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const u2 w = {codes4(x[e][0], x[e][1], x[e][2], x[e][3], ik), codes4(x[e][4], x[e][5], x[e][6], x[e][7], ik)};
          *reinterpret_cast<u2 *>(Kp + (keep + t) * D + (e ? d.hi : d.lo)) = bad ? u2{0x7f7f7f7fu, 0x7f7f7f7fu} : w;
        }
      };
      auto put_v = [&](int it, const float (&x)[4][4]) {  // 16 bytes; those of slots that are not new stay
        const int g = g0 + it / D4, t0 = 4 * g - keep;
        u4 *dst = reinterpret_cast<u4 *>(Vp + (g * D + it % D4 * 4) * 4);
        uint32_t row[4], fresh = 0;  // the codes of a slot's four dims
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool is_new = t0 + r >= 0 && t0 + r < nt;
          row[r] = is_new && !bad_token[t0 + r] ? codes4(x[r][0], x[r][1], x[r][2], x[r][3], iv) : 0;
          fresh |= is_new ? 0xffu << (8 * r) : 0;
        }
        u4 w = {0, 0, 0, 0};
        if (fresh != 0xffffffffu) w = *dst;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t c = ((row[0] >> (8 * e)) & 0xffu) | (((row[1] >> (8 * e)) & 0xffu) << 8) |
                             (((row[2] >> (8 * e)) & 0xffu) << 16) | (((row[3] >> (8 * e)) & 0xffu) << 24);
          w[e] = (w[e] & ~fresh) | c;
        }
        *dst = w;
      };
      // where the scale grows, the kept tokens' codes first (a group of four slots may hold kept and new ones)
      if (keep && ek > eko) {
        const float f = exp2i(eko - ek);  // no less than 2^-120
        for (int it = tid; it < keep * (D / 8); it += nthr) {
          u2 *dst = reinterpret_cast<u2 *>(Kp) + it;
          *dst = u2{recode4(dst->x, f), recode4(dst->y, f)};
        }
      }
      if (keep && ev > evo) {
        const float f = exp2i(evo - ev);
        for (int it = tid; it < ((keep + 3) >> 2) * D4; it += nthr) {
          u4 *dst = reinterpret_cast<u4 *>(Vp) + it;
          const int left = keep - it / D4 * 4;
          const uint32_t m = left >= 4 ? 0xffffffffu : (1u << (8 * left)) - 1;
          u4 w = *dst;
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = (recode4(w[e], f) & m) | (w[e] & ~m);
          *dst = w;
        }
        __syncthreads();
      }
      if (tid < nk) put_k(tid, kx);
      if (tid < nv) put_v(tid, vx);
      for (int it = tid + nthr; it < nk; it += nthr) {
        float x[2][8];
        load_k(it, x);
        put_k(it, x);
      }
      for (int it = tid + nthr; it < nv; it += nthr) {
        float x[4][4];
        load_v(it, x);
        put_v(it, x);
      }
    }
    if (!a.per_seq) break;
    __syncthreads();  // bad_token and red are the next page's
  }
}

template <int DT>
static void launch_append(int D, const KvAppendArgs &a, dim3 grid, int threads, hipStream_t s) {
  switch (D) {
    case 64: hipLaunchKernelGGL((k_kv_append<DT, 64>), grid, dim3(threads), 0, s, a); break;
    case 128: hipLaunchKernelGGL((k_kv_append<DT, 128>), grid, dim3(threads), 0, s, a); break;
    case 192: hipLaunchKernelGGL((k_kv_append<DT, 192>), grid, dim3(threads), 0, s, a); break;
    default: hipLaunchKernelGGL((k_kv_append<DT, 256>), grid, dim3(threads), 0, s, a); break;
  }
}

}  // namespace vybdq

using namespace vybdq;

extern "C" int vybdq_kv_append(uint64_t K, uint64_t V, uint64_t Ks, uint64_t Vs, int64_t n_pages, int64_t Hkv, int64_t D,
                               int64_t page, uint64_t k, uint64_t v, uint64_t q, uint64_t q_out, int x_dt, int64_t ldk,
                               int64_t ldv, int64_t ldq, int64_t Hq, uint64_t cosv, uint64_t sinv, int64_t R,
                               int64_t n_pos, int interleaved, uint64_t table, int64_t W, uint64_t q_start,
                               uint64_t ctx, int64_t T, int64_t B, int64_t max_new, uint64_t stream) {
  VYBDQ_REQUIRE(dt_valid_in(x_dt), VYBDQ_ERR_ARG, "x_dt must be F32, F16 or BF16");
  VYBDQ_REQUIRE(D == 64 || D == 128 || D == 192 || D == 256, VYBDQ_ERR_SHAPE, "D must be 64, 128, 192 or 256");
  VYBDQ_REQUIRE(page >= 16 && page <= 256 && (page & (page - 1)) == 0, VYBDQ_ERR_SHAPE,
                "page must be a power of two in 16 .. 256");
  VYBDQ_REQUIRE(n_pages >= 1 && n_pages < (int64_t(1) << 31), VYBDQ_ERR_SHAPE, "n_pages must be in 1 .. 2^31 - 1");
  VYBDQ_REQUIRE(Hkv >= 1 && Hkv <= 1024, VYBDQ_ERR_SHAPE, "Hkv must be in 1 .. 1024");
  VYBDQ_REQUIRE(T >= 0 && T < (int64_t(1) << 30) && B >= 0 && B < (int64_t(1) << 20), VYBDQ_ERR_SHAPE,
                "T must be below 2^30 and B below 2^20");
  VYBDQ_REQUIRE(W >= 1 && W * page < (int64_t(1) << 31), VYBDQ_ERR_SHAPE, "W must be at least 1 and W * page below 2^31");
  VYBDQ_REQUIRE(R >= 0 && R <= D && R % 16 == 0, VYBDQ_ERR_SHAPE, "R must be a multiple of 16 in 0 .. D");
  VYBDQ_REQUIRE(!q || (Hq >= Hkv && Hq % Hkv == 0 && Hq <= 16384), VYBDQ_ERR_SHAPE, "Hq must be a multiple of Hkv");
  // (a grid holds less than 2^32 threads along x)
  VYBDQ_REQUIRE((T / page + 2 * B) * Hkv < (int64_t(1) << 23), VYBDQ_ERR_SHAPE, "(T / page + 2 B) Hkv must be below 2^23");
  if (T == 0 || B == 0) return VYBDQ_OK;
  VYBDQ_REQUIRE(K && V && Ks && Vs && k && v && table && q_start && ctx, VYBDQ_ERR_ARG, "null pointer");
  VYBDQ_REQUIRE(!q || q_out, VYBDQ_ERR_ARG, "q needs q_out");
  VYBDQ_REQUIRE(R == 0 || (cosv && sinv && n_pos >= 1), VYBDQ_ERR_ARG, "a rotation needs cos and sin");
  const int es = dt_size(x_dt);
  VYBDQ_REQUIRE(ldk >= Hkv * D && ldv >= Hkv * D && (!q || ldq >= Hq * D), VYBDQ_ERR_SHAPE,
                "a row stride is smaller than a row");
  VYBDQ_REQUIRE((K | V | k | v | q | q_out | cosv | sinv) % 16 == 0 && ldk * es % 16 == 0 && ldv * es % 16 == 0 &&
                    (!q || ldq * es % 16 == 0),
                VYBDQ_ERR_ALIGN, "codes, rows, cos and sin must be 16-byte aligned");
  VYBDQ_REQUIRE((Ks | Vs | table | q_start | ctx) % 4 == 0, VYBDQ_ERR_ALIGN,
                "scales, table, q_start and ctx must be 4-byte aligned");
  KvAppendArgs a{};
  int ps = 4;
  while ((1 << ps) < page) ++ps;
  a.c = {reinterpret_cast<uint8_t *>(K), reinterpret_cast<uint8_t *>(V), reinterpret_cast<float *>(Ks),
         reinterpret_cast<float *>(Vs), static_cast<int32_t>(n_pages), static_cast<int32_t>(Hkv), ps};
  a.b = {reinterpret_cast<const int32_t *>(table), reinterpret_cast<const int32_t *>(q_start),
         reinterpret_cast<const int32_t *>(ctx), nullptr, W, static_cast<int32_t>(T), static_cast<int32_t>(B)};
  a.k = reinterpret_cast<const void *>(k);
  a.v = reinterpret_cast<const void *>(v);
  a.q = reinterpret_cast<const void *>(q);
  a.q_out = reinterpret_cast<void *>(q_out);
  a.cosv = reinterpret_cast<const float *>(cosv);
  a.sinv = reinterpret_cast<const float *>(sinv);
  a.ldk = ldk;
  a.ldv = ldv;
  a.ldq = ldq;
  a.G = q ? static_cast<int32_t>(Hq / Hkv) : 0;
  a.R = static_cast<int32_t>(R);
  a.n_pos = static_cast<int32_t>(n_pos < INT32_MAX ? n_pos : INT32_MAX);
  a.inter = interleaved != 0;
  a.per_seq = max_new == 1;
  const int64_t units = a.per_seq ? B : (T >> ps) + 2 * B;
  const int rc = kv_status_address(a.b.status);
  if (rc) return rc;
  // threads: a page's pieces of 16 dims (a decode step's 8 to 16: one wave, so that all workgroups of a batch are resident);
  // query heads: one turn of a piece to a thread
  const int64_t rows = max_new >= 1 && max_new < page ? max_new : T < page ? T : page;
  const int threads = rows * (D / 16) <= 64 ? 64 : rows * (D / 16) <= 256 ? 256 : 512;
  const int64_t q_wgs = q ? (rows * ((a.G + kv_turn_heads(x_dt) - 1) / kv_turn_heads(x_dt)) * (D / 16) + threads - 1) / threads : 0;
  const dim3 grid(static_cast<unsigned>(units * Hkv), static_cast<unsigned>(1 + (q_wgs < 64 ? q_wgs : 64)));
  hipStream_t s = as_stream(stream);
  VYBDQ_DISPATCH_IN(x_dt, DT, launch_append<DT>(static_cast<int>(D), a, grid, threads, s));
  return check_launch("vybdq_kv_append");
}

extern "C" int vybdq_kv_status(void) {
  uint32_t *st = nullptr;
  const int rc = kv_status_address(st);
  if (rc) return rc;
  uint32_t v = 0;
  hipError_t e = hipDeviceSynchronize();
  if (e == hipSuccess) {
    std::lock_guard<std::mutex> lock(g_kv_mu);  // (the word that k_kv_status_take leaves is this call's until it is read)
    hipLaunchKernelGGL(k_kv_status_take, dim3(1), dim3(1), 0, nullptr, st);
    e = hipGetLastError();
    if (e == hipSuccess) e = hipMemcpy(&v, st + 1, 4, hipMemcpyDeviceToHost);
  }
  if (e != hipSuccess) return set_error(VYBDQ_ERR_HIP, std::string("vybdq_kv_status: ") + hipGetErrorString(e));
  if (v & kKvBadRows) return set_error(VYBDQ_ERR_SHAPE, "q_start was not a rising sequence within the rows");
  if (v & kKvBadCtx) return set_error(VYBDQ_ERR_SHAPE, "a sequence's ctx was below its rows or past its pages");
  if (v & kKvBadPage) return set_error(VYBDQ_ERR_SHAPE, "a page of the table was outside the cache");
  if (v & kKvBadAngle) return set_error(VYBDQ_ERR_SHAPE, "a position was past the rows of cos and sin");
  return VYBDQ_OK;
}
