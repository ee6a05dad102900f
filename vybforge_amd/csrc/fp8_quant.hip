// Activations to e4m3 codes with a power-of-two scale per row and 128 columns (fp8.h), gfx950.
//
// 16 lanes take a block: 8 elements each (16 bytes of a 16-bit type), the block's largest magnitude by four DPP steps over
// the bits of |x| (an integer maximum: infinities and NaN come out on top), 8 codes a lane.
// Bound by memory: 8192 x 6144 bf16 25 us, 6.1 TB/s; one row of 6144 2.1 us, a launch and one wait for memory.
#include "fp8_load.h"

namespace vybdq {

template <int DT>
__global__ void __launch_bounds__(256) k_fp8_quant(const void *__restrict__ X, uint8_t *__restrict__ Xq,
                                                   float *__restrict__ Xs, uint32_t blocks, uint32_t KB, int K,
                                                   int64_t ldx) {
  const uint32_t u = blockIdx.x * 16u + (threadIdx.x >> 4);
  if (u >= blocks) return;  // (whole rows of 16 lanes leave)
  const uint32_t m = u / KB, b = u - m * KB;
  const int k = static_cast<int>(b) * 128 + static_cast<int>(threadIdx.x & 15) * 8;
  float x[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = 0.f;
  const bool in = k < K;
  if (in) fp8_load8<DT>(X, static_cast<int64_t>(m) * ldx + k, x);
  float sc;
  const u2 c = fp8_quant8(x, sc);
  if (in) *reinterpret_cast<u2 *>(Xq + static_cast<int64_t>(m) * K + k) = c;
  if ((threadIdx.x & 15) == 0) Xs[u] = sc;
}

// M ceil(K / 128) is at most kFp8QuantBlocks (the callers check)
int fp8_quant_rows(const void *X, int x_dt, int64_t M, int64_t K, int64_t ldx, uint8_t *Xq, float *Xs, hipStream_t s) {
  const int64_t KB = (K + 127) / 128, blocks = M * KB;
  const dim3 grid(static_cast<unsigned>((blocks + 15) / 16));
  VYBDQ_DISPATCH_IN(x_dt, DT, hipLaunchKernelGGL((k_fp8_quant<DT>), grid, dim3(256), 0, s, X, Xq, Xs,
                                                 static_cast<uint32_t>(blocks), static_cast<uint32_t>(KB),
                                                 static_cast<int>(K), ldx));
  return check_launch("fp8 quantizer");
}

}  // namespace vybdq

using namespace vybdq;

extern "C" int vybdq_quant_fp8(uint64_t X, int x_dt, int64_t ldx, uint64_t Xq, uint64_t Xs, int64_t M, int64_t K,
                               uint64_t stream) {
  VYBDQ_REQUIRE(dt_valid_in(x_dt), VYBDQ_ERR_ARG, "x_dt must be F32, F16 or BF16");
  VYBDQ_REQUIRE(M >= 0 && K >= 16 && K % 16 == 0 && K < (int64_t(1) << 23), VYBDQ_ERR_SHAPE,
                "M must not be negative, K must be a multiple of 16 in 16 .. 2^23 - 16");
  VYBDQ_REQUIRE(M <= kFp8QuantBlocks && M * ((K + 127) / 128) <= kFp8QuantBlocks, VYBDQ_ERR_SHAPE,
                "M ceil(K / 128) must be at most 2^28 - 16");
  if (M == 0) return VYBDQ_OK;
  VYBDQ_REQUIRE(X && Xq && Xs, VYBDQ_ERR_ARG, "null buffer");
  VYBDQ_REQUIRE(M == 1 || ldx >= K, VYBDQ_ERR_SHAPE, "ldx is smaller than a row");
  VYBDQ_REQUIRE((X | Xq) % 16 == 0 && (M == 1 || ldx * dt_size(x_dt) % 16 == 0) && Xs % 4 == 0, VYBDQ_ERR_ALIGN,
                "rows of X and Xq must be 16-byte aligned, Xs 4-byte");
  const Fp8Span x{X, M, K * dt_size(x_dt), ldx * dt_size(x_dt)}, xq = fp8_bytes(Xq, M * K), xs = fp8_bytes(Xs, M * ((K + 127) / 128) * 4);
  VYBDQ_REQUIRE(!fp8_overlap(x, xq) && !fp8_overlap(x, xs) && !fp8_overlap(xq, xs), VYBDQ_ERR_ARG, "X, Xq and Xs must not overlap");
  return fp8_quant_rows(reinterpret_cast<const void *>(X), x_dt, M, K, ldx, reinterpret_cast<uint8_t *>(Xq),
                        reinterpret_cast<float *>(Xs), as_stream(stream));
}
