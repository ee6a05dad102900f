// Few rows of X times an e4m3 matrix: W streamed once from memory into registers, gfx950.
//
// A workgroup takes 16 rows of W and all rows of X (up to 16); its NW waves deal the K blocks among themselves (wave w: blocks w, w + NW,
// ..), so that together they read a row's bytes in order, and each sums its blocks' products in registers; the waves' sums are
// added through LDS in wave order. A wave asks for D blocks of W at once and has no wait but for them: D 16 128 bytes
// in flight to a wave.
//   LDSX: X comes as x_dt and is quantized (fp8.h) by every workgroup for itself into LDS, while its first loads of W are on their
//     way; otherwise X is codes and scales in memory, read like W (from L2).
// The product: fp8_mm.h (16 x 16 x 128 instructions; columns past the rows of X compute what nothing reads).
#pragma once

#include "fp8_mm.h"
#include "fp8_load.h"

namespace vybdq {

// One row's 16-byte chunk q of LDS codes: blocks of 128 bytes, the chunks of a block at chunk ^ (row & 7).
__device__ __forceinline__ int rows_chunk(int row, int q, int KB) { return (row * KB + (q >> 3)) * 128 + (((q & 7) ^ (row & 7)) * 16); }

// Quantize rows 0 .. M - 1 of X (row r at X + r ldx elements) into LDS: codes (rows_chunk) and scales [M][KB]. Chunks
// past K are zeros. All threads of the workgroup; no barrier.
template <int DT>
__device__ __forceinline__ void rows_quant(const void *X, int64_t ldx, int M, int K, int KB, char *codes, float *scales) {
  const int sub = threadIdx.x & 15, step = blockDim.x >> 4;  // 16 lanes to a block of 128
  const int n = M * KB;
  for (int u = threadIdx.x >> 4; u < n; u += step) {
    const int r = u / KB, b = u - r * KB, k = b * 128 + sub * 8;
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = 0.f;
    if (k < K) fp8_load8<DT>(X, static_cast<int64_t>(r) * ldx + k, x);
    float sc;
    const u2 c = fp8_quant8(x, sc);
    *reinterpret_cast<u2 *>(codes + rows_chunk(r, b * 8 + (sub >> 1), KB) + 8 * (sub & 1)) = c;
    if (sub == 0) scales[u] = sc;
  }
}

struct Fp8RowsArgs {
  Fp8MmArgs m;
  const void *x;  // LDSX: X as x_dt
  int64_t ldx;
};

template <int NW, int D, int XDT, bool HALF>
__global__ void __launch_bounds__(64 * NW) k_fp8_rows(const Fp8RowsArgs ra) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr bool LDSX = XDT >= 0;
  const Fp8MmArgs &a = ra.m;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int g = lane >> 4, r16 = lane & 15;
  const int nk = a.KB, n0 = blockIdx.x * 16;
  const int tail = a.K & 127;
  // LDS: the waves' sums, then (LDSX) scales and codes of X
  f4 *red = reinterpret_cast<f4 *>(smem);
  float *xs_lds = reinterpret_cast<float *>(smem + NW * 1024);
  char *x_lds = smem + NW * 1024 + (a.M * nk * 4 + 127) / 128 * 128;

  const uint8_t *wp = a.W + static_cast<int64_t>(min(n0 + r16, a.N - 1)) * a.K;
  const float *wsp = a.Ws + static_cast<int64_t>(n0 >> 7) * nk;
  const int xrow = min(r16, a.M - 1);
  const uint8_t *xp = LDSX ? nullptr : a.X + static_cast<int64_t>(xrow) * a.K;
  const float *xsp = LDSX ? nullptr : a.Xs + xrow * a.xs_row;
  auto frag = [&](const uint8_t *p, int k) {  // the lane's two chunks of block k; zeros past the row's end
    const bool last = tail && k == nk - 1;
    const bool in0 = !last || 16 * g < tail, in1 = !last || 64 + 16 * g < tail;
    const uint8_t *q = p + static_cast<int64_t>(k) * 128;
    u4 c0 = *reinterpret_cast<const u4 *>(q + (in0 ? 16 * g : 0)), c1 = *reinterpret_cast<const u4 *>(q + (in1 ? 64 + 16 * g : 0));
    if (last) {
      c0 = in0 ? c0 : u4{0, 0, 0, 0};
      c1 = in1 ? c1 : u4{0, 0, 0, 0};
    }
    i8v f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[j] = static_cast<int>(c0[j]);
      f[4 + j] = static_cast<int>(c1[j]);
    }
    return f;
  };
  f4 acc = {0.f, 0.f, 0.f, 0.f};
  bool ready = !LDSX;
  for (int k0 = wave; k0 < nk || !ready; k0 += NW * D) {
    i8v wf[D];
    float ws[D];
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int k = k0 + NW * d;
      if (k < nk) {
        wf[d] = frag(wp, k);
        ws[d] = uniform_load(wsp, k);
      }
    }
    if constexpr (LDSX) {
      if (!ready) {
        rows_quant<XDT < 0 ? 0 : XDT>(ra.x, ra.ldx, a.M, a.K, nk, x_lds, xs_lds);
        __syncthreads();
        ready = true;
      }
    }
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int k = k0 + NW * d;
      if (k >= nk) break;
      i8v xf;
      float xs;
      if constexpr (LDSX) {
        const u4 c0 = *reinterpret_cast<const u4 *>(x_lds + rows_chunk(xrow, 8 * k + g, nk));
        const u4 c1 = *reinterpret_cast<const u4 *>(x_lds + rows_chunk(xrow, 8 * k + 4 + g, nk));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          xf[j] = static_cast<int>(c0[j]);
          xf[4 + j] = static_cast<int>(c1[j]);
        }
        xs = xs_lds[xrow * nk + k];
      } else {
        xf = frag(xp, k);
        xs = xsp[k];
      }
      const f4 t = fp8_block<HALF>(wf[d], xf);
      const float s = xs * ws[d];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = fmaf(t[i], s, acc[i]);
    }
  }
  red[wave * 64 + lane] = acc;
  __syncthreads();
  if (wave == 0) {  // the sum over the waves
    f4 s = red[lane];
#pragma unroll
    for (int w = 1; w < NW; ++w) s += red[w * 64 + lane];
    const int col = n0 + 4 * g, left = r16 < a.M ? a.N - col : 0;
    const int64_t at = static_cast<int64_t>(r16) * a.ldy + col;
    switch (a.ydt) {
      case VYBDQ_F32: fp8_put4<VYBDQ_F32>(a, at, left, s); break;
      case VYBDQ_F16: fp8_put4<VYBDQ_F16>(a, at, left, s); break;
      case VYBDQ_BF16: fp8_put4<VYBDQ_BF16>(a, at, left, s); break;
      default: fp8_put4<VYBDQ_F64>(a, at, left, s); break;
    }
  }
}

// LDS of a launch: the waves' sums, and X's scales and codes where they are made there
inline int64_t fp8_rows_lds(int NW, bool ldsx, int64_t M, int64_t KB) {
  return NW * 1024 + (ldsx ? (M * KB * 4 + 127) / 128 * 128 + M * KB * 128 : 0);
}

template <int NW, int D, int XDT, bool HALF>
int fp8_rows_launch(const Fp8RowsArgs &a, hipStream_t s) {
  const int64_t lds = fp8_rows_lds(NW, XDT >= 0, a.m.M, a.m.KB);
  static std::atomic<uint64_t> raised{0};
  auto *fn = &k_fp8_rows<NW, D, XDT, HALF>;
  if (lds > 64 * 1024) {
    const int rc = ensure_lds_limit(reinterpret_cast<const void *>(fn), 160 * 1024, raised, "fp8 product (few rows)");
    if (rc) return rc;
  }
  hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>((a.m.N + 15) / 16)), dim3(64 * NW), lds, s, a);
  return check_launch("fp8 product (few rows)");
}

}  // namespace vybdq
