// The product of e4m3 matrices (fp8_mm.h) as a GEMM, and with the quantizer in front as a linear layer, gfx950.
#include "fp8_rows.h"

#include <cstdio>
#include <cstdlib>

namespace vybdq {

// Sums of a split product: Y = RS + the splits' float32 sums in order, four elements to a thread.
__global__ void __launch_bounds__(256) k_fp8_join(const Fp8MmArgs a, const float *__restrict__ part, int64_t stride, int splits) {
  const int64_t i4 = 4 * (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x);
  const int64_t n4 = (a.N + 3) / 4 * 4;
  const int64_t row = i4 / n4;
  const int col = static_cast<int>(i4 - row * n4);
  if (row >= a.M) return;
  const int left = a.N - col;
  const float *p = part + row * a.N + col;
  f4 v = {0.f, 0.f, 0.f, 0.f};
  if (a.N % 4 == 0) {
    for (int s = 0; s < splits; ++s) v += *reinterpret_cast<const f4 *>(p + s * stride);
  } else {
    for (int s = 0; s < splits; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < left) v[j] += p[s * stride + j];
  }
  const int64_t at = row * a.ldy + col;
  switch (a.ydt) {
    case VYBDQ_F32: fp8_put4<VYBDQ_F32>(a, at, left, v); break;
    case VYBDQ_F16: fp8_put4<VYBDQ_F16>(a, at, left, v); break;
    case VYBDQ_BF16: fp8_put4<VYBDQ_BF16>(a, at, left, v); break;
    default: fp8_put4<VYBDQ_F64>(a, at, left, v); break;
  }
}

// ---- which kernel ---------------------------------------------------------------------------------

struct Fp8Plan {
  int BM, splits;  // pipelined tiles of BM x 256 (64, 128, 192, 256); BM = 0: the forms for any K
};

constexpr int64_t kFp8PartBytes = int64_t(64) << 20;  // most bytes of float32 sums that a split product writes

// Bytes of split sums that a call of M rows may use: rises with M, so that a workspace serves every smaller batch.
static int64_t fp8_part_bytes(int64_t M, int64_t N, int64_t K) {
  const int64_t one = M * N * 4, most = (K + 127) / 128 / 4;  // (no split of fewer than 4 blocks)
  if (most < 2 || M > 1024) return 0;
  const int64_t n = one * (most < 16 ? most : 16);
  return n < kFp8PartBytes ? n : kFp8PartBytes;
}

// Tile height and splits with the least estimate: rounds of tiles over the chip, a round its K steps and its end; split sums written,
// read and added. Times in us fitted over 26 shapes from 16 to 2048 rows (both instructions) with every tile and up to 16 splits
// forced: 9% off in the mean over 200 of them, the choice never more than 2% above the best of them; with the tiles of 192 rows
// (512 x 17408 x 5120 62 us, the others 68 to 81; 2048 rows 176 / 207), 11 more shapes up to 4096 rows: at most 5% (4096 x 9728 x 2560
// 131 us, 124 with 128 rows). A K that ends inside a block: 512 x 17408 x 5136 84 us with the same estimate.
static Fp8Plan fp8_plan(int64_t M, int64_t N, int64_t K, bool half, int64_t part) {
  const int64_t nk = (K + 127) / 128, cus = device_cu_count();
  Fp8Plan best{0, 1};
  if (nk < 4) return best;
  constexpr double kStep[2][4] = {{0.84, 1.0, 1.25, 1.72}, {1.07, 1.65, 0, 0}}, kEnd[4] = {2.5, 2.8, 2.9, 2.9};
  double best_t = 1e30;
  for (int c = 0; c < (half ? 2 : 4); ++c) {
    if (c == 2 && K % 128) continue;  // (that tile has no registers left for a short block)
    const int BM = 64 * (c + 1);
    const int64_t tiles = (M + BM - 1) / BM * ((N + 255) / 256);
    for (int64_t S = 1; S <= 16; ++S) {
      if (S > 1 && (nk / S < 4 || S * M * N * 4 > part)) break;
      const double rounds = static_cast<double>((tiles * S + cus - 1) / cus);
      const double t = rounds * (static_cast<double>((nk + S - 1) / S) * kStep[half][c] + kEnd[c]) +
                       (S > 1 ? 3.2 + static_cast<double>(S * M * N) * 8 / 4.5e6 : 0.0);
      if (t < best_t) best_t = t, best = Fp8Plan{BM, static_cast<int>(S)};
    }
  }
  if (const char *e = tuning_env("VYBDQ_FP8_TILE")) {  // "BM,splits"
    int bm = 0, sp = 0;
    if (sscanf(e, "%d,%d", &bm, &sp) == 2 && (bm == 64 || bm == 128 || (((bm == 192 && K % 128 == 0) || bm == 256) && !half)) && sp >= 1 && nk / sp >= 4 &&
        (sp == 1 || sp * M * N * 4 <= part))
      best = Fp8Plan{bm, sp};
  }
  return best;
}

// Few rows of X (fp8_rows.h) or tiles. Up to 4 rows, or 16 of at most 2^25 weights, the streaming form is the faster one (measured,
// bf16: 1 x 17408 x 5120 22.3 us against 23.8, 1 x 2560 x 9728 10.0 / 15.2, 16 x 9728 x 2560 11.5 / 13.5); beyond, every
// workgroup's own pass over X costs more than the tiles' second launch (16 x 17408 x 5120 32.8 / 25.0, 16 x 5120 x 17408 42 / 26).
static bool fp8_rows_take(int64_t M, int64_t N, int64_t K) { return M <= 4 || (M <= 16 && (N * K <= (int64_t(1) << 25) || K < 512)); }

// Whether such a call quantizes X in its workgroups, each for itself: where that is little beside its rows of W, or all
// workgroups do it at once (measured with the quantizer's own launch: 1 x 9728 x 2560 8.3 us against 11.0, 4 x 17408 x 5120
// 25.1 / 26.4, 16 x 1003 x 2560 8.2 / 10.3; but 16 x 9728 x 2560 17.0 / 13.5). Its codes and scales fit with two workgroups to a CU.
static bool fp8_rows_quant(int64_t M, int64_t N, int64_t K) {
  return (M <= 4 || N <= 4096) && M * ((K + 127) / 128) * 132 <= 56 * 1024;
}

// 16 waves from 32 blocks of K, else 8 (1 x 2560 x 9728 10.0 us against 12.0; 1 x 6144 x 2048 9.5 / 8.9).
template <int XDT, bool HALF>
static int fp8_rows_run(const Fp8RowsArgs &r, hipStream_t s) {
  return r.m.KB >= 32 ? fp8_rows_launch<16, 3, XDT, HALF>(r, s) : fp8_rows_launch<8, 3, XDT, HALF>(r, s);
}

template <bool HALF, bool TAIL>
static int fp8_pipe_run(int BM, const Fp8MmArgs &t, int64_t n, hipStream_t s) {
  if (BM == 64) return fp8_pipe_launch<4, 2, 1, 8, 3, FP8_DENSE, HALF, TAIL>(t, n, s);
  if constexpr (!HALF) {
    if (BM == 256) return fp8_pipe_launch<8, 4, 2, 4, 2, FP8_DENSE, false, TAIL>(t, n, s);
    if constexpr (!TAIL)
      if (BM == 192) return fp8_pipe_launch<6, 4, 2, 4, 2, FP8_DENSE, false>(t, n, s);
  }
  return fp8_pipe_launch<4, 4, 2, 4, 3, FP8_DENSE, HALF, TAIL>(t, n, s);
}

template <bool HALF>
static int fp8_gemm_tiles(Fp8MmArgs &a, float *part, int64_t part_bytes, hipStream_t s) {
  auto units = [&](int BM, int BN) {
    a.m_tiles = (a.M + BM - 1) / BM;
    a.n_tiles = (a.N + BN - 1) / BN;
    const int64_t n = static_cast<int64_t>(a.m_tiles) * a.n_tiles * a.splits;
    a.units = static_cast<int>(n);
    return n;
  };
  a.splits = 1;
  const int64_t allowed = fp8_part_bytes(a.M, a.N, a.K);
  if (fp8_rows_take(a.M, a.N, a.K)) {
    Fp8RowsArgs r{};
    r.m = a;
    return fp8_rows_run<-1, HALF>(r, s);
  }
  const Fp8Plan p = fp8_plan(a.M, a.N, a.K, HALF, part && part_bytes >= allowed ? allowed : 0);
  if (p.BM) {
    Fp8MmArgs t = a;
    t.splits = p.splits;
    if (p.splits > 1) {
      t.Y = part;
      t.ydt = VYBDQ_F32;
      t.ldy = a.N;
      t.RS = nullptr;
      t.wide = a.N % 4 == 0;
      t.split_stride = static_cast<int64_t>(a.M) * a.N;
    }
    a.splits = p.splits;
    const int64_t n = units(p.BM, 256);
    t.m_tiles = a.m_tiles;
    t.n_tiles = a.n_tiles;
    t.units = a.units;
    const int rc = a.K % 128 ? fp8_pipe_run<HALF, true>(p.BM, t, n, s) : fp8_pipe_run<HALF, false>(p.BM, t, n, s);
    if (rc || p.splits == 1) return rc;
    const int64_t threads = static_cast<int64_t>(a.M) * ((a.N + 3) / 4);
    hipLaunchKernelGGL(k_fp8_join, dim3(static_cast<unsigned>((threads + 255) / 256)), dim3(256), 0, s, a, part, t.split_stride, p.splits);
    return check_launch("fp8 product (join)");
  }
  if (a.M <= 64) return fp8_mm_launch<4, 2, 1, 4, 3, FP8_DENSE, HALF>(a, units(64, 128), s);
  if (a.M <= 512) return fp8_mm_launch<4, 4, 2, 2, 2, FP8_DENSE, HALF>(a, units(128, 128), s);
  return fp8_mm_launch<8, 4, 2, 4, 2, FP8_DENSE, HALF>(a, units(256, 256), s);
}

static Fp8MmArgs fp8_args(const uint8_t *W, const float *Ws, const uint8_t *Xq, const float *Xs, void *Y, int y_dt, int64_t M,
                          int64_t N, int64_t K, int64_t ldy, const void *RS) {
  Fp8MmArgs a{};
  a.X = Xq;
  a.Xs = Xs;
  a.W = W;
  a.Ws = Ws;
  a.M = static_cast<int>(M);
  a.N = static_cast<int>(N);
  a.K = static_cast<int>(K);
  a.KB = static_cast<int>((K + 127) / 128);
  a.xs_row = a.KB;
  a.x_rows = M;
  a.Y = Y;
  a.ydt = y_dt;
  a.ldy = ldy;
  a.RS = RS;
  const int64_t es = 4 * dt_size(y_dt);
  a.wide = N % 4 == 0 && ldy % 4 == 0 && (reinterpret_cast<uint64_t>(Y) | reinterpret_cast<uint64_t>(RS)) % es == 0;
  return a;
}

// float32 outputs keep float32 sums. Those of 16 bits take the e4m3 instruction, at 1.76 times the rate (library products of 8192^3:
// 2568 against 1456 TFLOP/s; 4096 x 17408 x 5120 389 us, float32 631): it drops 1.4e-5 of a sum's rms for normal data and 6e-5 where
// a few columns of X are thirty times the others, beside roundings of 2.1e-4 (float16: the error against 64 bits grows by
// 2 to 4%) and 1.7e-3 (bfloat16: by 0.05%), and never more than the bound in fp8_mm.h. Codes are 2^-4 of their values off themselves.
static bool fp8_half(int y_dt) { return y_dt == VYBDQ_F32 || y_dt == VYBDQ_F64; }

static int fp8_gemm(Fp8MmArgs a, float *part, int64_t part_bytes, hipStream_t s) {
  return fp8_half(a.ydt) ? fp8_gemm_tiles<true>(a, part, part_bytes, s) : fp8_gemm_tiles<false>(a, part, part_bytes, s);
}

}  // namespace vybdq

using namespace vybdq;

static int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }

static int fp8_check(const char *func, int64_t M, int64_t N, int64_t K, uint64_t W, uint64_t Ws, uint64_t Y, int y_dt,
                     int64_t &ldy, uint64_t RS) {
  auto bad = [&](int code, const char *msg) { return set_error(code, std::string(func) + ": " + msg); };
  if (!dt_valid_out(y_dt)) return bad(VYBDQ_ERR_ARG, "y_dt must be F32, F16, BF16 or F64");
  if (K < 16 || K % 16 || K >= (int64_t(1) << 23)) return bad(VYBDQ_ERR_SHAPE, "K must be a multiple of 16 in 16 .. 2^23 - 16");
  if (N < 1 || N >= (int64_t(1) << 24) || M < 0 || M >= (int64_t(1) << 24))
    return bad(VYBDQ_ERR_SHAPE, "N must be in 1 .. 2^24 - 1 and M below 2^24");
  if ((M + 127) / 128 * ((N + 127) / 128) >= (int64_t(1) << 22)) return bad(VYBDQ_ERR_SHAPE, "ceil(M / 128) ceil(N / 128) must be below 2^22");
  if (ldy == 0) ldy = N;
  if (ldy < N) return bad(VYBDQ_ERR_SHAPE, "ldy is smaller than a row");
  if (M == 0) return VYBDQ_OK;
  if (!W || !Ws || !Y) return bad(VYBDQ_ERR_ARG, "null buffer");
  if (W % 16) return bad(VYBDQ_ERR_ALIGN, "W must be 16-byte aligned");
  if (Ws % 4 || Y % dt_size(y_dt) || RS % dt_size(y_dt)) return bad(VYBDQ_ERR_ALIGN, "Ws, Y and RS must be aligned to their elements");
  return VYBDQ_OK;
}

// Y and the workspace are written while workgroups still read everything else; RS may be Y itself, whose elements are read by the
// thread that writes them.
static int fp8_check_overlap(const char *func, int64_t M, int64_t N, int64_t K, uint64_t W, uint64_t Ws, uint64_t Y, int y_dt,
                             int64_t ldy, uint64_t RS, const Fp8Span &ws, std::initializer_list<Fp8Span> x) {
  auto bad = [&](const char *msg) { return set_error(VYBDQ_ERR_ARG, std::string(func) + ": " + msg); };
  const Fp8Span y{Y, M, N * dt_size(y_dt), ldy * dt_size(y_dt)}, rs{RS, M, y.width, y.pitch};
  const Fp8Span w = fp8_bytes(W, N * K), s = fp8_bytes(Ws, (N + 127) / 128 * ((K + 127) / 128) * 4);
  for (const Fp8Span &in : x) {
    if (fp8_overlap(y, in)) return bad("Y must not overlap X: workgroups read X while others write");
    if (fp8_overlap(ws, in)) return bad("the workspace must not overlap X");
  }
  if (fp8_overlap(y, w) || fp8_overlap(y, s)) return bad("Y must not overlap W or Ws");
  if (RS != Y && fp8_overlap(y, rs)) return bad("RS must be Y or not overlap it");
  if (fp8_overlap(ws, w) || fp8_overlap(ws, s) || fp8_overlap(ws, y) || fp8_overlap(ws, rs))
    return bad("the workspace must not overlap W, Ws, Y or RS");
  return VYBDQ_OK;
}

extern "C" int64_t vybdq_gemm_fp8_workspace_size(int64_t M, int64_t N, int64_t K) {
  if (M < 0 || M >= (int64_t(1) << 24) || N < 1 || N >= (int64_t(1) << 24) || K < 16 || K % 16 || K >= (int64_t(1) << 23)) return -1;
  return align256(fp8_part_bytes(M < 1024 ? M : 1024, N, K));  // (rises with M, none above 1024)
}

extern "C" int vybdq_gemm_fp8(uint64_t W, uint64_t Ws, uint64_t Xq, uint64_t Xs, uint64_t Y, int64_t M, int64_t N, int64_t K,
                              int y_dt, int64_t ldy, uint64_t RS, uint64_t ws, int64_t ws_bytes, uint64_t stream) {
  const int rc = fp8_check(__func__, M, N, K, W, Ws, Y, y_dt, ldy, RS);
  if (rc || M == 0) return rc;
  VYBDQ_REQUIRE(Xq && Xs, VYBDQ_ERR_ARG, "null buffer");
  VYBDQ_REQUIRE(Xq % 16 == 0 && Xs % 4 == 0, VYBDQ_ERR_ALIGN, "Xq must be 16-byte and Xs 4-byte aligned");
  VYBDQ_REQUIRE(ws % 256 == 0 && ws_bytes >= 0, VYBDQ_ERR_WORKSPACE, "workspace must be 256-byte aligned");
  const int64_t part = fp8_part_bytes(M, N, K), used = ws && ws_bytes >= part ? part : 0;
  const int orc = fp8_check_overlap(__func__, M, N, K, W, Ws, Y, y_dt, ldy, RS, fp8_bytes(ws, used),
                                    {fp8_bytes(Xq, M * K), fp8_bytes(Xs, M * ((K + 127) / 128) * 4)});
  if (orc) return orc;
  return fp8_gemm(fp8_args(reinterpret_cast<const uint8_t *>(W), reinterpret_cast<const float *>(Ws),
                           reinterpret_cast<const uint8_t *>(Xq), reinterpret_cast<const float *>(Xs), reinterpret_cast<void *>(Y),
                           y_dt, M, N, K, ldy, reinterpret_cast<const void *>(RS)),
                  reinterpret_cast<float *>(ws), ws_bytes, as_stream(stream));
}

extern "C" int64_t vybdq_linear_fp8_workspace_size(int64_t M, int64_t N, int64_t K) {
  const int64_t part = vybdq_gemm_fp8_workspace_size(M, N, K);
  return part < 0 ? -1 : align256(M * K) + align256(M * ((K + 127) / 128) * 4) + part;
}

extern "C" int vybdq_linear_fp8(uint64_t W, uint64_t Ws, uint64_t X, int x_dt, int64_t ldx, uint64_t Y, int64_t M, int64_t N,
                                int64_t K, int y_dt, int64_t ldy, uint64_t RS, uint64_t ws, int64_t ws_bytes, uint64_t stream) {
  VYBDQ_REQUIRE(dt_valid_in(x_dt), VYBDQ_ERR_ARG, "x_dt must be F32, F16 or BF16");
  const int rc = fp8_check(__func__, M, N, K, W, Ws, Y, y_dt, ldy, RS);
  if (rc || M == 0) return rc;
  VYBDQ_REQUIRE(X, VYBDQ_ERR_ARG, "null buffer");
  VYBDQ_REQUIRE(M * ((K + 127) / 128) <= kFp8QuantBlocks, VYBDQ_ERR_SHAPE, "M ceil(K / 128) must be at most 2^28 - 16");
  VYBDQ_REQUIRE(M == 1 || ldx >= K, VYBDQ_ERR_SHAPE, "ldx is smaller than a row");
  VYBDQ_REQUIRE(X % 16 == 0 && (M == 1 || ldx * dt_size(x_dt) % 16 == 0), VYBDQ_ERR_ALIGN, "rows of X must be 16-byte aligned");
  VYBDQ_REQUIRE(ws && ws % 256 == 0 && ws_bytes >= vybdq_linear_fp8_workspace_size(M, N, K), VYBDQ_ERR_WORKSPACE,
                "workspace must be 256-byte aligned and of vybdq_linear_fp8_workspace_size bytes");
  const int orc = fp8_check_overlap(__func__, M, N, K, W, Ws, Y, y_dt, ldy, RS, fp8_bytes(ws, vybdq_linear_fp8_workspace_size(M, N, K)),
                                    {Fp8Span{X, M, K * dt_size(x_dt), ldx * dt_size(x_dt)}});
  if (orc) return orc;
  uint8_t *xq = reinterpret_cast<uint8_t *>(ws);
  float *xs = reinterpret_cast<float *>(ws + align256(M * K));
  const int64_t front = align256(M * K) + align256(M * ((K + 127) / 128) * 4);
  hipStream_t s = as_stream(stream);
  const Fp8MmArgs a = fp8_args(reinterpret_cast<const uint8_t *>(W), reinterpret_cast<const float *>(Ws), xq, xs,
                               reinterpret_cast<void *>(Y), y_dt, M, N, K, ldy, reinterpret_cast<const void *>(RS));
  if (fp8_rows_take(M, N, K) && fp8_rows_quant(M, N, K)) {
    const Fp8RowsArgs r{a, reinterpret_cast<const void *>(X), ldx};
    if (fp8_half(y_dt)) VYBDQ_DISPATCH_IN(x_dt, XDT, return (fp8_rows_run<XDT, true>(r, s)))
    else VYBDQ_DISPATCH_IN(x_dt, XDT, return (fp8_rows_run<XDT, false>(r, s)))
  }
  const int qc = fp8_quant_rows(reinterpret_cast<const void *>(X), x_dt, M, K, ldx, xq, xs, s);
  if (qc) return qc;
  return fp8_gemm(a, reinterpret_cast<float *>(ws + front), ws_bytes - front, s);
}
