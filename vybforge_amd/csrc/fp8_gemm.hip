// The product of e4m3 matrices (fp8_mm.h) as a GEMM, and with the quantizer in front as a linear layer, gfx950.
#include "fp8_mm.h"

namespace vybdq {

template <bool HALF>
static int fp8_gemm_tiles(Fp8MmArgs &a, hipStream_t s) {
  auto units = [&](int BM, int BN) {
    a.m_tiles = (a.M + BM - 1) / BM;
    a.n_tiles = (a.N + BN - 1) / BN;
    const int64_t n = static_cast<int64_t>(a.m_tiles) * a.n_tiles;
    a.units = static_cast<int>(n);
    return n;
  };
  if (a.M <= 16) return fp8_mm_launch<1, 2, 1, 4, 4, FP8_DENSE, HALF>(a, units(16, 128), s);
  if (a.M <= 64) return fp8_mm_launch<4, 2, 1, 4, 3, FP8_DENSE, HALF>(a, units(64, 128), s);
  if (a.K % 128 == 0 && a.KB >= 4 && a.M > 64) {
    if (a.M <= 128) return fp8_pipe_launch<4, 2, 2, 4, 4, FP8_DENSE, HALF>(a, units(128, 128), s);
    if (HALF || a.M <= 512) return fp8_pipe_launch<4, 4, 2, 4, 3, FP8_DENSE, HALF>(a, units(128, 256), s);
    return fp8_pipe_launch<8, 4, 2, 4, 2, FP8_DENSE, false>(a, units(256, 256), s);
  }
  if (a.M <= 512) return fp8_mm_launch<4, 4, 2, 2, 2, FP8_DENSE, HALF>(a, units(128, 128), s);
  return fp8_mm_launch<8, 4, 2, 4, 2, FP8_DENSE, HALF>(a, units(256, 256), s);
}

static int fp8_gemm(const uint8_t *W, const float *Ws, const uint8_t *Xq, const float *Xs, void *Y, int y_dt, int64_t M,
                    int64_t N, int64_t K, int64_t ldy, const void *RS, hipStream_t s) {
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
  a.xs_block = 1;
  a.x_rows = M;
  a.Y = Y;
  a.ydt = y_dt;
  a.ldy = ldy;
  a.RS = RS;
  const int64_t es = 4 * dt_size(y_dt);
  a.wide = N % 4 == 0 && ldy % 4 == 0 && (reinterpret_cast<uint64_t>(Y) | reinterpret_cast<uint64_t>(RS)) % es == 0;
  // float32 outputs keep float32 sums; those of 16 bits round by more than the e4m3 instruction loses
  return y_dt == VYBDQ_F32 || y_dt == VYBDQ_F64 ? fp8_gemm_tiles<true>(a, s) : fp8_gemm_tiles<false>(a, s);
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

extern "C" int vybdq_gemm_fp8(uint64_t W, uint64_t Ws, uint64_t Xq, uint64_t Xs, uint64_t Y, int64_t M, int64_t N, int64_t K,
                              int y_dt, int64_t ldy, uint64_t RS, uint64_t stream) {
  const int rc = fp8_check(__func__, M, N, K, W, Ws, Y, y_dt, ldy, RS);
  if (rc || M == 0) return rc;
  VYBDQ_REQUIRE(Xq && Xs, VYBDQ_ERR_ARG, "null buffer");
  VYBDQ_REQUIRE(Xq % 16 == 0 && Xs % 4 == 0, VYBDQ_ERR_ALIGN, "Xq must be 16-byte and Xs 4-byte aligned");
  return fp8_gemm(reinterpret_cast<const uint8_t *>(W), reinterpret_cast<const float *>(Ws), reinterpret_cast<const uint8_t *>(Xq),
                  reinterpret_cast<const float *>(Xs), reinterpret_cast<void *>(Y), y_dt, M, N, K, ldy,
                  reinterpret_cast<const void *>(RS), as_stream(stream));
}

extern "C" int64_t vybdq_linear_fp8_workspace_size(int64_t M, int64_t N, int64_t K) {
  if (M < 0 || M >= (int64_t(1) << 24) || N < 1 || N >= (int64_t(1) << 24) || K < 16 || K % 16 || K >= (int64_t(1) << 23)) return -1;
  return align256(M * K) + align256(M * ((K + 127) / 128) * 4);
}

extern "C" int vybdq_linear_fp8(uint64_t W, uint64_t Ws, uint64_t X, int x_dt, int64_t ldx, uint64_t Y, int64_t M, int64_t N,
                                int64_t K, int y_dt, int64_t ldy, uint64_t RS, uint64_t ws, int64_t ws_bytes, uint64_t stream) {
  VYBDQ_REQUIRE(dt_valid_in(x_dt), VYBDQ_ERR_ARG, "x_dt must be F32, F16 or BF16");
  const int rc = fp8_check(__func__, M, N, K, W, Ws, Y, y_dt, ldy, RS);
  if (rc || M == 0) return rc;
  VYBDQ_REQUIRE(X, VYBDQ_ERR_ARG, "null buffer");
  VYBDQ_REQUIRE(M * ((K + 127) / 128) < (int64_t(1) << 28), VYBDQ_ERR_SHAPE, "M ceil(K / 128) must be below 2^28");
  VYBDQ_REQUIRE(M == 1 || ldx >= K, VYBDQ_ERR_SHAPE, "ldx is smaller than a row");
  VYBDQ_REQUIRE(X % 16 == 0 && (M == 1 || ldx * dt_size(x_dt) % 16 == 0), VYBDQ_ERR_ALIGN, "rows of X must be 16-byte aligned");
  VYBDQ_REQUIRE(ws && ws % 256 == 0 && ws_bytes >= vybdq_linear_fp8_workspace_size(M, N, K), VYBDQ_ERR_WORKSPACE,
                "workspace must be 256-byte aligned and of vybdq_linear_fp8_workspace_size bytes");
  uint8_t *xq = reinterpret_cast<uint8_t *>(ws);
  float *xs = reinterpret_cast<float *>(ws + align256(M * K));
  const int qc = fp8_quant_rows(reinterpret_cast<const void *>(X), x_dt, M, K, ldx, xq, xs, as_stream(stream));
  if (qc) return qc;
  return fp8_gemm(reinterpret_cast<const uint8_t *>(W), reinterpret_cast<const float *>(Ws), xq, xs, reinterpret_cast<void *>(Y),
                  y_dt, M, N, K, ldy, reinterpret_cast<const void *>(RS), as_stream(stream));
}
