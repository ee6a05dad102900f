// 8-bit floating-point matrices: e4m3 codes with a float32 scale for each block of 128 x 128 weights, and for each row
// and 128 columns of activations. What the quantizer (fp8_quant.hip), the products (fp8_mm.h) and the experts
// (moe_fp8.hip) share.
//
//   weight W[n, k] = code * Ws[n / 128][k / 128]      activation X[m, k] = code * Xs[m][k / 128]
//   Xs = 2^e with the least e in [-100, 120] for which every |x| of the block is at most 448 * 2^e (448: the largest e4m3);
//   code = e4m3(x * 2^-e), ties to even: the product with a power of two is exact, so a code is x rounded once. A block that
//   holds an infinity or NaN has the scale NaN (and zero codes): exactly the rows of the product that it takes part in are NaN.
#pragma once

#include "common.h"

#include <initializer_list>
#include <type_traits>
#include <utility>

namespace vybdq {

constexpr int kFp8ExpMin = -100, kFp8ExpMax = 120;

typedef int i8v __attribute__((ext_vector_type(8)));

__device__ __forceinline__ float fp8_exp2(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// The exponent of a block whose largest |x| has the bits `u` (finite): 448 = 1.75 * 2^8.
__device__ __forceinline__ int fp8_exponent(uint32_t u) {
  const int x = static_cast<int>(u >> 23) - 127, e = (u & 0x7fffffu) <= 0x600000u ? x - 8 : x - 7;
  return e < kFp8ExpMin ? kFp8ExpMin : (e > kFp8ExpMax ? kFp8ExpMax : e);
}

// A block's scale and the factor of its codes from the bits of its largest |x|.
__device__ __forceinline__ float fp8_scale(uint32_t amax, float &inv) {
  if (amax >= 0x7f800000u) {
    inv = 0.f;
    return __uint_as_float(0x7fc00000u);
  }
  const int e = fp8_exponent(amax);
  inv = fp8_exp2(-e);
  return fp8_exp2(e);
}

// Four values of a block times the power of two that its scale divides by, as e4m3 codes, rounded to nearest even (none is
// above 448 then). Zeros where inv = 0: the block holds an infinity or NaN.
__device__ __forceinline__ uint32_t fp8_codes4(float a, float b, float c, float d, float inv) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false);
  const uint32_t v = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, lo, true));
  return inv == 0.f ? 0u : v;
}

// Largest 32-bit value over the 16 lanes of a row, in every lane (DPP, on the VALU).
__device__ __forceinline__ uint32_t row16_max_u32(uint32_t v) {
  auto step = [&](auto ctrl) {
    const uint32_t o = static_cast<uint32_t>(
        __builtin_amdgcn_update_dpp(0, static_cast<int>(v), decltype(ctrl)::value, 0xf, 0xf, false));
    v = o > v ? o : v;
  };
  step(std::integral_constant<int, DPP_QUAD_XOR1>{});
  step(std::integral_constant<int, DPP_QUAD_XOR2>{});
  step(std::integral_constant<int, DPP_HALF_MIRROR>{});
  step(std::integral_constant<int, DPP_ROW_MIRROR>{});
  return v;
}

// Rows of `width` bytes every `pitch` bytes from `at` on (width <= pitch).
struct Fp8Span {
  uint64_t at;
  int64_t rows, width, pitch;
};
inline Fp8Span fp8_bytes(uint64_t at, int64_t n) { return {at, 1, n, n}; }

// Whether two buffers share a byte: exact, so that neighbouring columns of one wider matrix pass.
inline bool fp8_overlap(Fp8Span a, Fp8Span b) {
  for (Fp8Span *s : {&a, &b})
    if (s->rows == 1 || s->pitch == s->width) *s = fp8_bytes(s->at, s->rows * s->width);
  auto size = [](const Fp8Span &s) { return s.width > 0 ? static_cast<uint64_t>((s.rows - 1) * s.pitch + s.width) : 0; };
  if (!a.at || !b.at || size(a) == 0 || size(b) == 0) return false;  // (0: not given)
  if (a.at >= b.at + size(b) || b.at >= a.at + size(a)) return false;
  if (a.rows == 1) std::swap(a, b);
  // one row of b: whether the first row of a that ends behind its start begins before its end
  auto row = [&](uint64_t at) {
    const int64_t d = static_cast<int64_t>(at - a.at), i = d < a.width ? 0 : (d - a.width) / a.pitch + 1;
    return i < a.rows && i * a.pitch < d + b.width;
  };
  if (b.rows == 1) return row(b.at);
  if (a.pitch == b.pitch) {  // b's row j begins d bytes into row j + q of a's pitch
    if (a.at > b.at) std::swap(a, b);
    const int64_t q = static_cast<int64_t>(b.at - a.at) / a.pitch, d = static_cast<int64_t>(b.at - a.at) % a.pitch;
    return (q < a.rows && d < a.width) || (q + 1 < a.rows && d + b.width > a.pitch);
  }
  for (int64_t j = 0; j < b.rows; ++j)
    if (row(b.at + static_cast<uint64_t>(j * b.pitch))) return true;
  return false;
}

constexpr int64_t kFp8QuantBlocks = (int64_t(1) << 28) - 16;  // most blocks of a quantizer's launch: 16 threads each, below 2^32 in all

int fp8_quant_rows(const void *X, int x_dt, int64_t M, int64_t K, int64_t ldx, uint8_t *Xq, float *Xs, hipStream_t s);

}  // namespace vybdq
