// The paged 8-bit key/value cache: its layout, the batch that one call works on, and what the kernels that
// write it (kv_append.hip) and read it (kv_attn.h) share.
//
// Cache of one layer: page p holds P consecutive tokens of one sequence (P = 16 .. 256, a power of two), for each
// of Hkv heads of D = 64, 128, 192 or 256 dims:
//   K e4m3 [n_pages][Hkv][P][D]: the token in slot s at row s.
//   V e4m3 [n_pages][Hkv][P / 4][D][4]: four tokens side by side per dim. The matrix instruction that forms P V
//     wants consecutive tokens of one dim in a lane; four tokens to a dword give it whole registers without a
//     transpose, and an append still touches 4 D consecutive bytes.
//   Ks, Vs float32 [n_pages][Hkv]: a power of two per page and head (value = code * scale).
// 16 tokens of a head are 16 D consecutive bytes of K and of V alike, so a page is a run of such blocks.
#pragma once

#include "common.h"

namespace vybdq {

constexpr int kKvExpMin = -60, kKvExpMax = 60;  // exponents of a page's scale
constexpr float kKvCodeMax = 448.0f;            // largest finite e4m3

// status bits (vybdq_kv_status)
constexpr uint32_t kKvBadRows = 1u, kKvBadCtx = 2u, kKvBadPage = 4u, kKvBadAngle = 8u;

int kv_status_address(uint32_t *&ptr);

struct KvCacheArgs {
  uint8_t *K, *V;
  float *Ks, *Vs;
  int32_t n_pages, Hkv, ps;  // P = 1 << ps
};

// Sequence b of B: rows q_start[b] .. q_start[b + 1] - 1 of q / k / v are its last tokens, ctx[b] its tokens with
// them, table[b * W + i] the page of its tokens i P .. i P + P - 1.
struct KvBatchArgs {
  const int32_t *table, *q_start, *ctx;
  uint32_t *status;
  int64_t W;
  int32_t T, B;
};

__device__ __forceinline__ void kv_flag(uint32_t *status, uint32_t bit) {
  __hip_atomic_fetch_or(status, bit, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The last b < B with first(b) <= u, for first non-decreasing and first(0) <= u: 64 candidates a round, one per
// lane (one round up to 64 sequences). Every lane of the wave has to take part; the result is wave-uniform and
// within 0 .. B - 1 whatever first returns.
template <class F>
__device__ __forceinline__ int kv_find(int B, int64_t u, F first) {
  const int lane = threadIdx.x & 63;
  int lo = 0, len = B;
  while (len > 1) {
    const int step = (len + 63) >> 6;
    const int at = lane * step;
    const int n = __popcll(__ballot(at < len && first(lo + at) <= u));
    const int skip = n > 0 ? (n - 1) * step : 0;
    lo += skip;
    len = len - skip < step ? len - skip : step;
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

struct KvSeq {
  int s0, n, ctx;  // first row, rows, tokens
  bool ok;
};

__device__ __forceinline__ KvSeq kv_seq(const KvBatchArgs &a, int b) {
  KvSeq q;
  q.s0 = a.q_start[b];
  const int s1 = a.q_start[b + 1];
  q.ctx = a.ctx[b];
  q.ok = q.s0 >= 0 && q.s0 <= s1 && s1 <= a.T;
  q.n = q.ok ? s1 - q.s0 : 0;
  if (!q.ok && (threadIdx.x & 63) == 0) kv_flag(a.status, kKvBadRows);
  return q;
}

}  // namespace vybdq
