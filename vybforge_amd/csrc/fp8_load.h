// Reading activations and quantizing eight neighbours of a block of 128 columns, 16 lanes to a block (fp8.h).
#pragma once

#include "fp8.h"

namespace vybdq {

template <int DT>
__device__ __forceinline__ void fp8_load8(const void *p, int64_t i, float (&x)[8]) {
  if constexpr (DT == VYBDQ_F32) {
    const f4 *q = reinterpret_cast<const f4 *>(static_cast<const float *>(p) + i);
    const f4 a = q[0], b = q[1];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = a[j];
      x[4 + j] = b[j];
    }
  } else {
    const u4 r = *reinterpret_cast<const u4 *>(static_cast<const uint16_t *>(p) + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t w = r[j];
      if constexpr (DT == VYBDQ_F16) {
        x[2 * j] = half_bits_to_f32(w & 0xffffu);
        x[2 * j + 1] = half_bits_to_f32(w >> 16);
      } else {
        x[2 * j] = __uint_as_float(w << 16);
        x[2 * j + 1] = __uint_as_float(w & 0xffff0000u);
      }
    }
  }
}

// This lane's eight codes of a block that the 16 lanes of its row hold (8 consecutive columns each), and the block's scale. The
// largest magnitude is an integer maximum over the bits of |x|: infinities and NaN come out on top.
__device__ __forceinline__ u2 fp8_quant8(const float (&x)[8], float &scale) {
  uint32_t a = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t v = __float_as_uint(x[j]) & 0x7fffffffu;
    a = v > a ? v : a;
  }
  a = row16_max_u32(a);
  float inv;
  scale = fp8_scale(a, inv);
  return u2{fp8_codes4(x[0], x[1], x[2], x[3], inv), fp8_codes4(x[4], x[5], x[6], x[7], inv)};
}

}  // namespace vybdq
