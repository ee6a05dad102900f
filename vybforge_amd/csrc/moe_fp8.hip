// Mixture-of-experts layer over e4m3 experts with block scales (fp8.h), gfx950.
//
//   router (route_groups.h) -> idx, w;  x -> codes and scales per token and 128 columns
//   expert e: a = silu(min(x Wg_e, L)) * clamp(x Wu_e, -L, L) in float32, then codes and scales per row and 128 columns
//             e_out = a Wd_e
//   out[t] = sum over s of w[t, s] e_out[idx[t, s]](t) + shared(x[t]), float32, rounded once to out_dt
//
// On the stream, no host synchronisation: quantizer, router, bucketing (rows by expert and the list of their m-tiles; the
// shared expert's rows and tiles are one more expert's), gate and up of all rows with the activation and its quantizer as
// epilogue (k_fp8_mm<.., FP8_GATE_UP>: float32 gate and up never leave registers), down (FP8_DOWN), the weighted sum.
#include "fp8_load.h"
#include "fp8_mm.h"
#include "route_groups.h"

namespace vybdq {

int64_t moe_tiles_bound(int64_t T, int64_t E, int64_t k, int64_t rows);

// Where rows and tiles go: pos (token, slot) -> row, row -> token, the list of m-tiles.
struct MoeFp8Lists {
  int *pos, *row_map, *ntiles;
  int4 *tiles;
};

// Few tokens (at most 8, and 64 rows) in one launch: workgroup 0 routes them and lists rows and tiles, the others quantize x (one
// token of 6144 over 256 experts: 7.1 to 8.3 us; quantizer, router and bucketing by themselves 2.0, 5.4 and 4.6, and two gaps).
template <bool SOFTMAX, bool BIAS, int TOP, int ENT>
__global__ void __launch_bounds__(256) k_moe_fp8_front(const RouteArgs r, const void *__restrict__ x, int x_dt, int H,
                                                       uint8_t *__restrict__ xq, float *__restrict__ xs, int BM, int shared,
                                                       const MoeFp8Lists l) {
  __shared__ int idx_lds[64];
  if (blockIdx.x == 0) {
    for (int t = threadIdx.x >> 6; t < r.T; t += 4) route_groups_wave<SOFTMAX, BIAS, TOP, ENT>(r, t, idx_lds);
    __syncthreads();
    if (threadIdx.x < 64) bucket_rows_wave(idx_lds, r.T, r.topk, BM, BM, shared, l.pos, l.row_map, l.tiles, l.ntiles, nullptr, nullptr);
    return;
  }
  const int64_t u = static_cast<int64_t>(blockIdx.x - 1) * 16 + (threadIdx.x >> 4);  // 16 lanes to a block of 128 (H is whole blocks)
  if (u >= static_cast<int64_t>(r.T) * (H >> 7)) return;
  const int64_t at = u * 128 + (threadIdx.x & 15) * 8;
  float v[8], sc;
  VYBDQ_DISPATCH_IN(x_dt, DT, fp8_load8<DT>(x, at, v));
  *reinterpret_cast<u2 *>(xq + at) = fp8_quant8(v, sc);
  if ((threadIdx.x & 15) == 0) xs[u] = sc;
}

// Many tokens, one workgroup: rows per expert, the first row and tile of each (thread e: expert e), then every (token, slot)'s row.
// A row's place among its expert's comes from an atomic cursor: no result depends on it, each row is computed from its own token
// alone and added through pos. One CU, so in proportion to the rows: 384 rows 4.6 us, 32768 rows 21 to 29 (70 with 256 threads).
__global__ void __launch_bounds__(1024) k_moe_fp8_bucket(const int *__restrict__ idx, int T, int topk, int E, int BM, int shared,
                                                         const MoeFp8Lists l) {
  __shared__ int cnt[1024], wave_rows[16], wave_tiles[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = T * topk;
  cnt[tid] = 0;
  __syncthreads();
  for (int i = tid; i < n; i += 1024) atomicAdd(&cnt[idx[i]], 1);
  __syncthreads();
  const int c = tid < E ? cnt[tid] : 0, mt = (c + BM - 1) / BM;
  int r = c, t = mt;  // inclusive sums over the wave, then over the waves before
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int a = __shfl_up(r, d), b = __shfl_up(t, d);
    r += lane >= d ? a : 0;
    t += lane >= d ? b : 0;
  }
  if (lane == 63) {
    wave_rows[wave] = r;
    wave_tiles[wave] = t;
  }
  __syncthreads();
  const int tsh = shared ? (T + BM - 1) / BM : 0;
  int r0 = r - c, t0 = tsh + t - mt;
  for (int w = 0; w < wave; ++w) {
    r0 += wave_rows[w];
    t0 += wave_tiles[w];
  }
  for (int m = 0; m < mt; ++m) l.tiles[t0 + m] = make_int4(tid, r0, r0 + c, m);
  if (tid == 1023) *l.ntiles = t0 + mt;
  cnt[tid] = r0;  // (this thread's own count was read above): the expert's cursor
  for (int j = tid; j < tsh; j += 1024) l.tiles[j] = make_int4(-1, n, n + T, j);
  if (shared)
    for (int i = tid; i < T; i += 1024) l.row_map[n + i] = i;
  __syncthreads();
  for (int i = tid; i < n; i += 1024) {
    const int p = atomicAdd(&cnt[idx[i]], 1);
    l.pos[i] = p;
    l.row_map[p] = i / topk;
  }
}

// out[t][h] = sum over s of w[t, s] rows[pos[t, s]][h] + shared[t][h] in slot order; four columns to a thread.
template <int ODT>
__global__ void __launch_bounds__(256) k_moe_fp8_sum(const float *__restrict__ rows, const float *__restrict__ shared,
                                                     const int *__restrict__ pos, const float *__restrict__ w, int64_t T,
                                                     int topk, int64_t H, void *__restrict__ out) {
  const int64_t i = 4 * (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x);
  if (i >= T * H) return;
  const int64_t t = i / H, h = i - t * H;
  f4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < topk; ++s) {
    const f4 v = *reinterpret_cast<const f4 *>(rows + static_cast<int64_t>(pos[t * topk + s]) * H + h);
    const float ws = w[t * topk + s];
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = fmaf(ws, v[j], acc[j]);
  }
  if (shared) acc += *reinterpret_cast<const f4 *>(shared + i);
#pragma unroll
  for (int j = 0; j < 4; ++j) store_elem<ODT>(out, nullptr, i + j, acc[j]);
}

struct MoeFp8Ws {
  int *idx, *pos, *row_map, *ntiles;
  int4 *tiles;
  float *w, *xs, *as, *rows;
  uint8_t *xq, *aq;
  int64_t bytes;
};

static MoeFp8Ws moe_fp8_layout(char *base, int64_t T, int64_t H, int64_t I, int64_t E, int64_t k) {
  MoeFp8Ws m{};
  int64_t off = 0;
  auto take = [&](int64_t n) {
    char *p = base ? base + off : nullptr;
    off += (n + 255) / 256 * 256;
    return p;
  };
  const int64_t R = T * k + T;  // rows, the shared expert's among them
  m.idx = reinterpret_cast<int *>(take(4 * T * k));
  m.w = reinterpret_cast<float *>(take(4 * T * k));
  m.pos = reinterpret_cast<int *>(take(4 * T * k));
  m.row_map = reinterpret_cast<int *>(take(4 * R));
  m.tiles = reinterpret_cast<int4 *>(take(16 * moe_tiles_bound(T, E, k, 16)));
  m.ntiles = reinterpret_cast<int *>(take(4));
  m.xq = reinterpret_cast<uint8_t *>(take(T * H));
  m.xs = reinterpret_cast<float *>(take(4 * T * (H / 128)));
  m.aq = reinterpret_cast<uint8_t *>(take(R * I));
  m.as = reinterpret_cast<float *>(take(4 * R * (I / 128)));
  m.rows = reinterpret_cast<float *>(take(4 * R * H));
  m.bytes = off;
  return m;
}

static bool moe_fp8_shape(int64_t T, int64_t H, int64_t I, int64_t E, int64_t k) {
  return T >= 0 && T < (1 << 20) && H >= 128 && H % 128 == 0 && H <= 65536 && I >= 128 && I % 128 == 0 && I <= 65536 && E >= 1 &&
         E <= 1024 && k >= 1 && k <= E && k <= 64 && T * k < (1 << 22) && T * H < (int64_t(1) << 32) &&
         moe_tiles_bound(T, E, k, 16) * ((H > I ? H : I) / 128) < (int64_t(1) << 22);  // (workgroups of a launch)
}

template <int MODE, bool HALF>
static int moe_fp8_mm(int BM, Fp8MmArgs &a, int64_t tiles, hipStream_t s) {
  a.n_tiles = MODE == FP8_GATE_UP ? a.N / 128 : (a.N + 255) / 256;
  const int64_t units = tiles * a.n_tiles;
  if (BM == 64 && a.KB >= 3) return fp8_pipe_launch<4, 2, 1, 8, 3, MODE, HALF>(a, units, s);
  if (BM == 128 && a.KB >= 3) return fp8_pipe_launch<4, 4, 2, 4, 3, MODE, HALF>(a, units, s);
  if (BM == 16) return fp8_mm_launch<1, 2, 1, 8, 4, MODE, HALF>(a, units, s);
  if (BM == 64) return fp8_mm_launch<4, 4, 1, 4, 3, MODE, HALF>(a, units, s);
  return fp8_mm_launch<4, 4, 2, 4, 3, MODE, HALF>(a, units, s);
}

}  // namespace vybdq

using namespace vybdq;

extern "C" int64_t vybdq_moe_fp8_workspace_size(int64_t T, int64_t H, int64_t I, int64_t E, int64_t topk) {
  return moe_fp8_shape(T, H, I, E, topk) ? moe_fp8_layout(nullptr, T, H, I, E, topk).bytes : -1;
}

extern "C" int vybdq_moe_forward_fp8(uint64_t x, int x_dt, uint64_t logits, int logits_dt, uint64_t bias, uint64_t gate,
                                     uint64_t gate_s, uint64_t up, uint64_t up_s, uint64_t down, uint64_t down_s,
                                     uint64_t sh_gate, uint64_t sh_gate_s, uint64_t sh_up, uint64_t sh_up_s, uint64_t sh_down,
                                     uint64_t sh_down_s, uint64_t out, int out_dt, uint64_t idx_out, uint64_t w_out, int64_t T,
                                     int64_t H, int64_t I, int64_t E, int64_t topk, double scale, double limit, int softmax,
                                     int renorm, int64_t groups, int64_t top_groups, int64_t group_top, uint64_t ws,
                                     int64_t ws_bytes, uint64_t stream) {
  VYBDQ_REQUIRE(dt_valid_in(x_dt), VYBDQ_ERR_ARG, "x_dt must be F32, F16 or BF16");
  VYBDQ_REQUIRE(dt_valid_in(out_dt), VYBDQ_ERR_ARG, "out_dt must be F32, F16 or BF16");
  VYBDQ_REQUIRE(moe_fp8_shape(T, H, I, E, topk), VYBDQ_ERR_SHAPE,
                "H and I must be multiples of 128 up to 65536, E up to 1024, topk up to 64, and not too many tokens");
  const bool shared = sh_gate != 0;
  VYBDQ_REQUIRE(shared == (sh_gate_s != 0) && shared == (sh_up != 0) && shared == (sh_up_s != 0) && shared == (sh_down != 0) &&
                    shared == (sh_down_s != 0),
                VYBDQ_ERR_ARG, "shared expert: give all three matrices with their scales or none");
  MoeFp8Ws m = moe_fp8_layout(reinterpret_cast<char *>(ws), T, H, I, E, topk);
  RouteArgs r;
  int rc = route_groups_args(__func__, r, logits, logits_dt, bias, idx_out ? idx_out : (ws ? reinterpret_cast<uint64_t>(m.idx) : 0),
                             w_out ? w_out : (ws ? reinterpret_cast<uint64_t>(m.w) : 0), ws || (idx_out && w_out) ? T : 0, E, topk,
                             scale, softmax, renorm, groups, top_groups, group_top);
  if (rc || T == 0) return rc;
  VYBDQ_REQUIRE(x && logits && gate && gate_s && up && up_s && down && down_s && out, VYBDQ_ERR_ARG, "null input or output");
  VYBDQ_REQUIRE(limit > 0, VYBDQ_ERR_ARG, "limit must be positive");
  VYBDQ_REQUIRE((x | gate | up | down | sh_gate | sh_up | sh_down | out) % 16 == 0 &&
                    (gate_s | up_s | down_s | sh_gate_s | sh_up_s | sh_down_s) % 4 == 0,
                VYBDQ_ERR_ALIGN, "x, out and codes must be 16-byte aligned, scales 4-byte");
  VYBDQ_REQUIRE(ws && ws % 256 == 0 && ws_bytes >= m.bytes, VYBDQ_ERR_WORKSPACE,
                "workspace must be 256-byte aligned and of vybdq_moe_fp8_workspace_size bytes");
  {
    // (x and logits have been read when out is written, so it may lie over them)
    const int64_t wb = I * H, sb = (I / 128) * (H / 128) * 4;
    Fp8Span in[15] = {fp8_bytes(x, T * H * dt_size(x_dt)), fp8_bytes(logits, T * E * dt_size(logits_dt)),
                      fp8_bytes(bias, 4 * E)};
    int n_in = 3;
    for (const uint64_t p : {gate, up, down}) in[n_in++] = fp8_bytes(p, E * wb);
    for (const uint64_t p : {gate_s, up_s, down_s}) in[n_in++] = fp8_bytes(p, E * sb);
    for (const uint64_t p : {sh_gate, sh_up, sh_down}) in[n_in++] = fp8_bytes(p, wb);
    for (const uint64_t p : {sh_gate_s, sh_up_s, sh_down_s}) in[n_in++] = fp8_bytes(p, sb);
    const Fp8Span o = fp8_bytes(out, T * H * dt_size(out_dt)), i = fp8_bytes(idx_out, 4 * T * topk), w = fp8_bytes(w_out, 4 * T * topk);
    const Fp8Span work = fp8_bytes(ws, m.bytes);
    bool alias = fp8_overlap(i, w);
    for (const Fp8Span &r : {o, i, w}) alias = alias || fp8_overlap(work, r);
    for (const Fp8Span &r : {i, w}) alias = alias || fp8_overlap(o, r);
    for (const Fp8Span &r : in) alias = alias || fp8_overlap(work, r) || fp8_overlap(i, r) || fp8_overlap(w, r);
    VYBDQ_REQUIRE(!alias, VYBDQ_ERR_ARG, "idx_out, w_out and the workspace must not overlap each other, out or an input");
  }
  hipStream_t s = as_stream(stream);
  // rows to a tile: 16 while the experts hit have 8 each in the mean, 128 from 64 on (256 experts of 6144 x 2048, 8 to a token: 48
  // tokens 968 us with 16, 1005 with 64; 512 tokens 1575 with 64, 1739 with 128; 2048 tokens 2560 / 2665; 2800 tokens 3070 / 2985;
  // 4096 tokens 4113 / 3909, with 192 rows 4150)
  const int64_t n = T * topk, hit = E < n ? E : n;
  const int BM = n <= 8 * hit ? 16 : n <= 64 * hit ? 64 : 128;
  const MoeFp8Lists lists{m.pos, m.row_map, m.ntiles, m.tiles};
  if (n <= 64 && T <= 8) {
    const dim3 grid(static_cast<unsigned>(1 + (T * (H / 128) + 15) / 16));
#define FRONT(SM, BI, TP, ENT)                                                                                                      \
  hipLaunchKernelGGL((k_moe_fp8_front<SM, BI, TP, ENT>), grid, dim3(256), 0, s, r, reinterpret_cast<const void *>(x), x_dt,             \
                     static_cast<int>(H), m.xq, m.xs, BM, shared ? 1 : 0, lists)
    VYBDQ_DISPATCH_ROUTE(r, FRONT)
#undef FRONT
    rc = check_launch("moe front");
  } else {
    rc = fp8_quant_rows(reinterpret_cast<const void *>(x), x_dt, T, H, H, m.xq, m.xs, s);
    if (rc) return rc;
    rc = route_groups_launch(r, s);
    if (rc) return rc;
    hipLaunchKernelGGL(k_moe_fp8_bucket, dim3(1), dim3(1024), 0, s, r.idx, static_cast<int>(T), static_cast<int>(topk), static_cast<int>(E),
                       BM, shared ? 1 : 0, lists);
    rc = check_launch("moe bucket");
  }
  if (rc) return rc;
  const int64_t tiles = moe_tiles_bound(T, E, topk, BM);
  Fp8MmArgs g{};
  g.X = m.xq;
  g.Xs = m.xs;
  g.W = reinterpret_cast<const uint8_t *>(gate);
  g.Ws = reinterpret_cast<const float *>(gate_s);
  g.W2 = reinterpret_cast<const uint8_t *>(up);
  g.W2s = reinterpret_cast<const float *>(up_s);
  g.Ss = reinterpret_cast<const uint8_t *>(sh_gate);
  g.Sss = reinterpret_cast<const float *>(sh_gate_s);
  g.S2 = reinterpret_cast<const uint8_t *>(sh_up);
  g.S2s = reinterpret_cast<const float *>(sh_up_s);
  g.N = static_cast<int>(I);
  g.K = static_cast<int>(H);
  g.KB = static_cast<int>(H / 128);
  g.xs_row = g.KB;
  g.x_rows = T;
  g.w_stride = I * H;
  g.ws_stride = (I / 128) * (H / 128);
  g.tiles = m.tiles;
  g.ntiles = m.ntiles;
  g.row_map = m.row_map;
  g.H = m.aq;
  g.Hs = m.as;
  g.limit = static_cast<float>(limit);
  // gate and up on fp16 instructions: what the e4m3 ones lose (1.4e-5 of a sum's rms) moves one activation in 5000 to the next
  // code, a hundredth of the output's rms and more where it is a large one (4096 tokens: 3.9 ms, with e4m3 instructions 2.9)
  rc = moe_fp8_mm<FP8_GATE_UP, true>(BM, g, tiles, s);
  if (rc) return rc;
  Fp8MmArgs d = g;
  d.X = m.aq;
  d.Xs = m.as;
  d.W = reinterpret_cast<const uint8_t *>(down);
  d.Ws = reinterpret_cast<const float *>(down_s);
  d.Ss = reinterpret_cast<const uint8_t *>(sh_down);
  d.Sss = reinterpret_cast<const float *>(sh_down_s);
  d.N = static_cast<int>(H);
  d.K = static_cast<int>(I);
  d.KB = static_cast<int>(I / 128);
  d.xs_row = d.KB;
  d.row_map = nullptr;
  d.Y = m.rows;
  d.ldy = H;
  // (down's sums are not quantized again: a 16-bit out takes the e4m3 instruction as a 16-bit Y of the product does)
  rc = out_dt == VYBDQ_F32 ? moe_fp8_mm<FP8_DOWN, true>(BM, d, tiles, s) : moe_fp8_mm<FP8_DOWN, false>(BM, d, tiles, s);
  if (rc) return rc;
  const float *sh = shared ? m.rows + n * H : nullptr;
  const unsigned grid = static_cast<unsigned>((T * H / 4 + 255) / 256);
  VYBDQ_DISPATCH_IN(out_dt, ODT, hipLaunchKernelGGL((k_moe_fp8_sum<ODT>), dim3(grid), dim3(256), 0, s, m.rows, sh, m.pos, r.w, T,
                                                    static_cast<int>(topk), H, reinterpret_cast<void *>(out)));
  return check_launch("moe sum");
}
