// Product of e4m3 activations and e4m3 weights with their block scales (fp8.h), gfx950:
//
//   Y[m, n] = RS[m, n] + sum over b of (Xs[m][b] Ws[n / 128][b]) * (sum over the block's k of X[m, k] W[n, k])
//
// The inner sum is one matrix instruction (16 x 16 x 128, from zero), the outer one a float32 fma per element: a float32
// scale of its own for every block cannot stay in the matrix core.
#pragma once

#include "fp8.h"

namespace vybdq {

enum { FP8_DENSE = 0, FP8_GATE_UP = 1, FP8_DOWN = 2 };

struct Fp8MmArgs {
  const uint8_t *X, *W, *W2;       // X [M][K]; W [N][K] (experts: of expert 0); W2: up (GATE_UP)
  const float *Xs, *Ws, *W2s;
  const uint8_t *Ss, *S2;          // the shared expert's W, W2
  const float *Sss, *S2s;
  int M, N, K, KB;
  int64_t w_stride, ws_stride;     // codes and scales from one expert to the next
  const int4 *tiles;               // {expert (-1: shared), first row, end row, m-tile of these rows}
  const int *ntiles, *row_map;     // row -> row of X (null: itself)
  int m_tiles, n_tiles, units;
  void *Y;
  int ydt;
  int64_t ldy;
  const void *RS;
  uint8_t *H;                      // GATE_UP: codes [rows][N] and scales [rows][N / 128] of the activation
  float *Hs;
  float limit;
};

// 16 zero bytes that lanes read where a row has ended inside a block
static __device__ const u4 kFp8Zero = {0, 0, 0, 0};

// 4 bytes a lane from global memory straight to LDS: lane L's to dst + 4 L (see lds_dma16)
__device__ __forceinline__ void lds_dma4(const void *src, const void *dst) {
  const uint32_t l = __builtin_amdgcn_readfirstlane(
      static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const void *)dst)));
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(src), "s"(l) : "memory", "m0");
}

// Four e4m3 codes' bytes of two dwords as eight fp16 values: exact (e4m3's range lies within fp16's normal one).
__device__ __forceinline__ h8 fp8_to_h8(int lo, int hi) {
  const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8(lo, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(lo, true);
  const f2 c = __builtin_amdgcn_cvt_pk_f32_fp8(hi, false), d = __builtin_amdgcn_cvt_pk_f32_fp8(hi, true);
  return h8{static_cast<_Float16>(a.x), static_cast<_Float16>(a.y), static_cast<_Float16>(b.x), static_cast<_Float16>(b.y),
            static_cast<_Float16>(c.x), static_cast<_Float16>(c.y), static_cast<_Float16>(d.x), static_cast<_Float16>(d.y)};
}

// The block product of 16 W rows (lane & 15) and 16 X rows (lane & 15): lane l's 32 bytes are chunks l >> 4 and 4 + (l >> 4)
// of its row's 128, for both operands alike, so each k meets its own. Result: n = 4 (l >> 4) + i, m = l & 15.
// HALF: on fp16 instructions, whose sums are those of float32. The e4m3 instruction aligns its products to the largest ones
// and loses what lies 2^-13 and more below them: 1.4e-5 (rms) of the block product's rms for normal data.
template <bool HALF>
__device__ __forceinline__ f4 fp8_block(const i8v &w, const i8v &x) {
  f4 t = {0.f, 0.f, 0.f, 0.f};
  if constexpr (HALF) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      t = __builtin_amdgcn_mfma_f32_16x16x32_f16(fp8_to_h8(w[2 * j], w[2 * j + 1]), fp8_to_h8(x[2 * j], x[2 * j + 1]), t, 0, 0, 0);
  } else {
    t = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, t, 0, 0, 0, 0, 0, 0);
  }
  return t;
}

// A float that is the same for the whole wave and that nothing writes during the launch: always a scalar load (a vector load
// would wait, in issue order, for every direct-to-LDS load behind it).
__device__ __forceinline__ float uniform_load(const float *p, int i) {
  return ((const float __attribute__((address_space(4))) *)p)[i];
}

template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Tiles of BM = 16 MF WM rows of X by BN = 16 NF WN rows of W, a K step of one block, WM x WN waves of 16 MF x 16 NF, both
// operands through LDS in ST stages by direct-to-LDS loads. A row's eight 16-byte chunks lie at chunk ^ (row & 7): the
// lanes of a read fall on distinct banks. A stage: X rows, W rows, the X rows' scales.
// Rows past the ends read the last one again (they reach only outputs that are not stored); chunks past K read zeros.
template <int MF, int NF, int WM, int WN, int ST, int MODE, bool HALF>
__global__ void __launch_bounds__(64 * WM * WN) k_fp8_mm(const Fp8MmArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int BM = 16 * MF * WM, BN = 16 * NF * WN, NW = WM * WN;
  constexpr int SB = (BM + 63) / 64 * 256, STAGE = (BM + BN) * 128 + SB;  // bytes of scales, of a stage
  constexpr int RL = (BM + BN) / 8;                                       // loads of 8 rows to a stage
  constexpr int PER = (RL + NW - 1) / NW, SPER = (BM / 64 + NW - 1) / NW > 0 ? (BM / 64 + NW - 1) / NW : 1;
  constexpr int LOADS = PER + SPER;  // a wave's loads to a stage
  constexpr bool DUAL = MODE == FP8_GATE_UP;
  static_assert(!DUAL || (BN == 256 && NF % 2 == 0), "a tile of gate and up holds one block of 128 columns of each");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int wm = wave / WN, wn = wave % WN;

  // the tile: rows [m0, m_end) of X (or of the row map), rows n0 .. of W
  int u = blockIdx.x, m0, m_end, n0;
  const uint8_t *W = a.W, *W2 = a.W2;
  const float *Ws = a.Ws, *W2s = a.W2s;
  if constexpr (MODE == FP8_DENSE) {
    if (a.units % 8 == 0) u = (u & 7) * (a.units >> 3) + (u >> 3);  // workgroups are dealt to the 8 XCDs in turn
    m0 = u % a.m_tiles * BM;
    n0 = u / a.m_tiles * BN;
    m_end = a.M;
  } else {
    const int t = u / a.n_tiles;
    if (t >= *a.ntiles) return;
    n0 = (u - t * a.n_tiles) * (DUAL ? 128 : BN);
    const int4 tile = a.tiles[t];
    m0 = tile.y + tile.w * BM;
    m_end = tile.z;
    if (tile.x < 0) {
      W = a.Ss;
      W2 = a.S2;
      Ws = a.Sss;
      W2s = a.S2s;
    } else {
      W += tile.x * a.w_stride;
      Ws += tile.x * a.ws_stride;
      if constexpr (DUAL) {
        W2 += tile.x * a.w_stride;
        W2s += tile.x * a.ws_stride;
      }
    }
  }

  // load j = wave + NW i of a stage: rows 8 j .. + 8 of the tile's X rows, then of its W rows
  const uint8_t *src[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    int j = wave + NW * i;
    if (j >= RL) j -= NW;  // (a load that is there already)
    const int r = 8 * j + (lane >> 3), c = (lane & 7) ^ (lane >> 3);
    const uint8_t *p;
    if (8 * j < BM) {
      int m = m0 + r < m_end ? m0 + r : m_end - 1;
      if (MODE != FP8_DENSE && a.row_map) m = a.row_map[m];
      p = a.X + static_cast<int64_t>(m) * a.K;
    } else if constexpr (DUAL) {
      // a wave's 16 NF rows: NF / 2 fragments of gate, then the same columns of up
      const int w = (r - BM) / (16 * NF), q = (r - BM) % (16 * NF);
      const int n = n0 + 8 * NF * w + q % (8 * NF);
      p = (q >= 8 * NF ? W2 : W) + static_cast<int64_t>(n) * a.K;
    } else {
      const int n = n0 + r - BM < a.N ? n0 + r - BM : a.N - 1;
      p = W + static_cast<int64_t>(n) * a.K;
    }
    src[i] = p + 16 * c;
  }
  const float *ssrc[SPER];
#pragma unroll
  for (int i = 0; i < SPER; ++i) {
    int m = m0 + ((wave + NW * i) * 64) % (SB / 4) + lane;
    m = m < m_end ? m : m_end - 1;
    if (MODE != FP8_DENSE && a.row_map) m = a.row_map[m];
    ssrc[i] = a.Xs + static_cast<int64_t>(m) * a.KB;
  }
  const int nk = a.KB, tail = a.K & 127;
  auto issue = [&](int k, char *buf) {
    const int c = (lane & 7) ^ (lane >> 3);
    const bool end = tail && k == nk - 1 && 16 * c >= tail;  // this lane's chunk lies behind the row
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      int j = wave + NW * i;
      if (j >= RL) j -= NW;
      const void *p = src[i] + 128 * static_cast<int64_t>(k);
      lds_dma16(end ? static_cast<const void *>(&kFp8Zero) : p, buf + 1024 * j);
    }
#pragma unroll
    for (int i = 0; i < SPER; ++i)
      lds_dma4(ssrc[i] + k, buf + (BM + BN) * 128 + ((wave + NW * i) * 256) % SB);
  };

  f4 acc[NF][MF];
#pragma unroll
  for (int n = 0; n < NF; ++n)
#pragma unroll
    for (int m = 0; m < MF; ++m) acc[n][m] = f4{0.f, 0.f, 0.f, 0.f};

  // this wave's scales of W: of n-block nb (and of the same block of up)
  const int nb = (DUAL ? n0 : min(n0 + 16 * NF * wn, a.N - 1)) >> 7;
  const float *wsp = Ws + static_cast<int64_t>(nb) * nk, *wsp2 = DUAL ? W2s + static_cast<int64_t>(nb) * nk : nullptr;
  static_assert(DUAL || 128 % (16 * NF) == 0, "a wave's rows of W lie in one block");
  const int lo = (lane & 15) * 128 + (((lane >> 4) ^ (lane & 7)) * 16);  // chunk lane >> 4; the other is at lo ^ 64
  const int xo = wm * 16 * MF * 128, wo = (BM + wn * 16 * NF) * 128, so = (BM + BN) * 128 + (wm * 16 * MF + (lane & 15)) * 4;
  auto frag = [&](const char *p) {
    const u4 p0 = *reinterpret_cast<const u4 *>(p + lo), p1 = *reinterpret_cast<const u4 *>(p + (lo ^ 64));
    i8v f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[j] = static_cast<int>(p0[j]);
      f[4 + j] = static_cast<int>(p1[j]);
    }
    return f;
  };
#pragma unroll
  for (int s = 0; s < ST - 1; ++s)
    if (s < nk) issue(s, smem + s * STAGE);
  float w0 = uniform_load(wsp, 0), w1 = DUAL ? uniform_load(wsp2, 0) : 0.f;
  for (int k = 0; k < nk; ++k) {
    const char *buf = smem + k % ST * STAGE;
    if (nk - k >= ST - 1) wait_loads<LOADS *(ST - 2)>();  // this wave's loads of stage k have arrived
    else wait_loads<0>();
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    if (k + ST - 1 < nk) issue(k + ST - 1, smem + (k + ST - 1) % ST * STAGE);  // every wave has left stage k - 1
    const int kn = k + 1 < nk ? k + 1 : k;
    const float w0n = uniform_load(wsp, kn), w1n = DUAL ? uniform_load(wsp2, kn) : 0.f;
    i8v wf[NF];
#pragma unroll
    for (int n = 0; n < NF; ++n) wf[n] = frag(buf + wo + 2048 * n);
#pragma unroll
    for (int m = 0; m < MF; ++m) {
      const i8v xf = frag(buf + xo + 2048 * m);
      const float xs = *reinterpret_cast<const float *>(buf + so + 64 * m);
      const float s0 = xs * w0, s1 = xs * w1;
#pragma unroll
      for (int n = 0; n < NF; ++n) {
        const f4 t = fp8_block<HALF>(wf[n], xf);
        const float sc = DUAL && n >= NF / 2 ? s1 : s0;
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[n][m][i] = fmaf(t[i], sc, acc[n][m][i]);
      }
    }
    w0 = w0n;
    w1 = w1n;
  }

  const int g4 = 4 * (lane >> 4);
  if constexpr (DUAL) {
    // acc[n][m]: gate of columns n0 + 8 NF wn + 16 n + g4 + i (n < NF / 2) and up of the same
    constexpr int HF = NF / 2;
    uint32_t top[MF];
#pragma unroll
    for (int m = 0; m < MF; ++m) {
      top[m] = 0;
#pragma unroll
      for (int n = 0; n < HF; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float g = acc[n][m][i], v = acc[HF + n][m][i];
          g = g > a.limit ? a.limit : g;  // (comparisons: a NaN stays)
          v = v > a.limit ? a.limit : (v < -a.limit ? -a.limit : v);
          const float e = __builtin_amdgcn_exp2f(g * -1.4426950408889634f);
          const float h = g * __builtin_amdgcn_rcpf(1.0f + e) * v;
          acc[n][m][i] = h;
          const uint32_t b = __float_as_uint(h) & 0x7fffffffu;
          top[m] = b > top[m] ? b : top[m];
        }
#pragma unroll
      for (int d = 16; d < 64; d <<= 1) {
        const uint32_t o = static_cast<uint32_t>(__shfl_xor(static_cast<int>(top[m]), d));
        top[m] = o > top[m] ? o : top[m];
      }
    }
    uint32_t *red = reinterpret_cast<uint32_t *>(smem);  // [WN][BM]
    __syncthreads();
    if (lane < 16)
#pragma unroll
      for (int m = 0; m < MF; ++m) red[wn * BM + (wm * MF + m) * 16 + lane] = top[m];
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MF; ++m) {
      const int r = (wm * MF + m) * 16 + (lane & 15);
      uint32_t t = 0;
#pragma unroll
      for (int w = 0; w < WN; ++w) t = red[w * BM + r] > t ? red[w * BM + r] : t;
      float inv;
      const float sc = fp8_scale(t, inv);
      const int row = m0 + r;
      if (row >= m_end) continue;
#pragma unroll
      for (int n = 0; n < HF; ++n) {
        const uint32_t c = fp8_codes4(acc[n][m][0], acc[n][m][1], acc[n][m][2], acc[n][m][3], inv);
        *reinterpret_cast<uint32_t *>(a.H + static_cast<int64_t>(row) * a.N + n0 + 8 * NF * wn + 16 * n + g4) = c;
      }
      if (wn == 0 && lane < 16) a.Hs[static_cast<int64_t>(row) * (a.N >> 7) + (n0 >> 7)] = sc;
    }
  } else {
#pragma unroll
    for (int m = 0; m < MF; ++m) {
      const int row = m0 + (wm * MF + m) * 16 + (lane & 15);
      if (row >= m_end) continue;
#pragma unroll
      for (int n = 0; n < NF; ++n) {
        const int col = n0 + 16 * (wn * NF + n) + g4;
        if constexpr (MODE == FP8_DOWN) {
          if (col < a.N) *reinterpret_cast<f4 *>(static_cast<float *>(a.Y) + static_cast<int64_t>(row) * a.ldy + col) = acc[n][m];
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (col + i >= a.N) continue;
            const int64_t at = static_cast<int64_t>(row) * a.ldy + col + i;
            const float v = acc[n][m][i];
            switch (a.ydt) {
              case VYBDQ_F32: store_elem<VYBDQ_F32>(a.Y, a.RS, at, v); break;
              case VYBDQ_F16: store_elem<VYBDQ_F16>(a.Y, a.RS, at, v); break;
              case VYBDQ_BF16: store_elem<VYBDQ_BF16>(a.Y, a.RS, at, v); break;
              default: store_elem<VYBDQ_F64>(a.Y, a.RS, at, v); break;
            }
          }
        }
      }
    }
  }
}

// Launch of one instantiation over `units` workgroups (below 2^22).
template <int MF, int NF, int WM, int WN, int ST, int MODE, bool HALF>
int fp8_mm_launch(const Fp8MmArgs &a, int64_t units, hipStream_t s) {
  constexpr int BM = 16 * MF * WM, BN = 16 * NF * WN, LDS = ST * ((BM + BN) * 128 + (BM + 63) / 64 * 256);
  static_assert(LDS <= 160 * 1024, "LDS");
  static std::atomic<uint64_t> raised{0};
  auto *fn = &k_fp8_mm<MF, NF, WM, WN, ST, MODE, HALF>;
  if (LDS > 64 * 1024) {
    const int rc = ensure_lds_limit(reinterpret_cast<const void *>(fn), LDS, raised, "fp8 product");
    if (rc) return rc;
  }
  hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(units)), dim3(64 * WM * WN), LDS, s, a);
  return check_launch("fp8 product");
}

}  // namespace vybdq
