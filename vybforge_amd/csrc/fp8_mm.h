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
  int64_t xs_row;                  // elements from one row's scales of X to the next's
  int64_t x_rows;                  // rows of X
  const uint8_t *Ss, *S2;          // the shared expert's W, W2
  const float *Sss, *S2s;
  int M, N, K, KB;
  int64_t w_stride, ws_stride;     // codes and scales from one expert to the next
  const int4 *tiles;               // {expert (-1: shared), first row, end row, m-tile of these rows}
  const int *ntiles, *row_map;     // row -> row of X (null: itself)
  int m_tiles, n_tiles, units;     // DENSE: units = tiles times splits of K
  int splits;
  int64_t split_stride;            // elements of Y from one split's sums to the next's (float32)
  void *Y;
  int ydt;
  int64_t ldy;
  const void *RS;
  int wide;                        // Y and RS: whole rows of aligned groups of four
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

// Eight e4m3 codes as fp16 values: exact (e4m3's range lies within fp16's normal one).
__device__ __forceinline__ h8 fp8_to_h8(int lo, int hi) {
  const h2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
  const h2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
  return h8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// The block product of 16 W rows (lane & 15) and 16 X rows (lane & 15): lane l's 32 bytes are chunks l >> 4 and 4 + (l >> 4)
// of its row's 128, for both operands alike, so each k meets its own. Result: n = 4 (l >> 4) + i, m = l & 15.
// HALF: on fp16 instructions, whose sums are those of float32. The e4m3 instruction takes eight neighbouring k (8 bytes of a lane)
// together and cuts, towards zero, each product below 2^-13 of the largest pair's 2^(exponent + exponent), where a subnormal
// code has the exponent -6 and a zero takes no part; the sums of eights add in float32. So it drops less than 7 * 2^-13 of the
// largest of eight: 1.4e-5 (rms) of the block product's rms for normal data, 2^-10 of sum |x w| at most with subnormal codes counted as
// 2^-6. (Sixteen eights whose large products cancel leave a sum that is off by 2^-6 of the largest.)
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

// Four neighbouring outputs, of which the first `left` exist, from element at on; a.wide: rows are whole and aligned groups of
// four.
template <int DT>
__device__ __forceinline__ void fp8_put4(const Fp8MmArgs &a, int64_t at, int left, const f4 &v) {
  if (left <= 0) return;
  if (a.wide && DT != VYBDQ_F64) {
    f4 o = v;
    if constexpr (DT == VYBDQ_F32) {
      if (a.RS) o += *reinterpret_cast<const f4 *>(static_cast<const float *>(a.RS) + at);
      *reinterpret_cast<f4 *>(static_cast<float *>(a.Y) + at) = o;
    } else if constexpr (DT == VYBDQ_F16) {
      if (a.RS) {
        const h4 r = *reinterpret_cast<const h4 *>(static_cast<const _Float16 *>(a.RS) + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] += static_cast<float>(r[i]);
      }
      h4 h;
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = static_cast<_Float16>(o[i]);
      *reinterpret_cast<h4 *>(static_cast<_Float16 *>(a.Y) + at) = h;
    } else {
      if (a.RS) {
        const u2 r = *reinterpret_cast<const u2 *>(static_cast<const uint16_t *>(a.RS) + at);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          o[2 * i] += __uint_as_float(r[i] << 16);
          o[2 * i + 1] += __uint_as_float(r[i] & 0xffff0000u);
        }
      }
      u2 b;
#pragma unroll
      for (int i = 0; i < 2; ++i) b[i] = f32_to_bf16(o[2 * i]) | (static_cast<uint32_t>(f32_to_bf16(o[2 * i + 1])) << 16);
      *reinterpret_cast<u2 *>(static_cast<uint16_t *>(a.Y) + at) = b;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < left) store_elem<DT>(a.Y, a.RS, at + i, v[i]);
}

// What becomes of a tile's sums: acc[n][m][i] is row m0 + 16 (WM m + wm) + (lane & 15), column n0 + 16 (NF wn + n) + 4 (lane / 16) + i
// (GATE_UP: fragments n < NF / 2 gate, the others up, of columns n0 + 8 NF wn + ..). red: LDS for WN x BM words (GATE_UP).
template <int MF, int NF, int WM, int WN, int MODE>
__device__ __forceinline__ void fp8_store(const Fp8MmArgs &a, f4 (&acc)[NF][MF], int m0, int m_end, int n0, uint32_t *red,
                                          int split = 0) {
  constexpr int BM = 16 * MF * WM;
  constexpr bool DUAL = MODE == FP8_GATE_UP;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int wm = wave / WN, wn = wave % WN;
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
          // (instructions of one ulp; the rounded product with log2 e makes |g| 2^-24 of it besides: 6e-7 of h at g = -10,
          // where h's code is 2^-4 of it off)
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
    __syncthreads();
    if (lane < 16)
#pragma unroll
      for (int m = 0; m < MF; ++m) red[wn * BM + (WM * m + wm) * 16 + lane] = top[m];
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MF; ++m) {
      const int r = (WM * m + wm) * 16 + (lane & 15);
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
  } else if constexpr (MODE == FP8_DOWN) {
#pragma unroll
    for (int m = 0; m < MF; ++m) {
      const int row = m0 + (WM * m + wm) * 16 + (lane & 15);
      if (row >= m_end) continue;
      float *y = static_cast<float *>(a.Y) + static_cast<int64_t>(row) * a.ldy;
#pragma unroll
      for (int n = 0; n < NF; ++n) {
        const int col = n0 + 16 * (wn * NF + n) + g4;
        if (col < a.N) *reinterpret_cast<f4 *>(y + col) = acc[n][m];
      }
    }
  } else {
    auto rows = [&](auto dt) {
      constexpr int DT = decltype(dt)::value;
#pragma unroll
      for (int m = 0; m < MF; ++m) {
        const int row = m0 + (WM * m + wm) * 16 + (lane & 15);
        const int64_t at = split * a.split_stride + static_cast<int64_t>(row) * a.ldy + n0 + 16 * wn * NF + g4;
#pragma unroll
        for (int n = 0; n < NF; ++n) {
          const int left = row < m_end ? a.N - (n0 + 16 * (wn * NF + n) + g4) : 0;
          fp8_put4<DT>(a, at + 16 * n, left, acc[n][m]);
          __builtin_amdgcn_sched_barrier(0);  // (a store's addresses at a time: registers)
        }
      }
    };
    switch (a.ydt) {
      case VYBDQ_F32: rows(std::integral_constant<int, VYBDQ_F32>{}); break;
      case VYBDQ_F16: rows(std::integral_constant<int, VYBDQ_F16>{}); break;
      case VYBDQ_BF16: rows(std::integral_constant<int, VYBDQ_BF16>{}); break;
      default: rows(std::integral_constant<int, VYBDQ_F64>{}); break;
    }
  }
}

// Unit u of the experts' tiles: its tile's list entry, column tile n and row tile m. The units of one expert take its row tiles
// side by side, columns by columns: they run at the same time on one XCD and share its W (4096 tokens over 256 experts of
// 6144 x 2048: the layer 4.07 ms with the tiles in list order, 3.9 so).
__device__ __forceinline__ int4 fp8_expert_unit(const Fp8MmArgs &a, int u, int BM, int &n, int &m) {
  const int t = u / a.n_tiles;
  const int4 q = a.tiles[t];
  const int c = (q.z - q.y + BM - 1) / BM, i = u - (t - q.w) * a.n_tiles;
  n = i / c;
  m = i - n * c;
  return q;
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
    if (u >= *a.ntiles * a.n_tiles) return;
    int n, m;
    const int4 tile = fp8_expert_unit(a, u, BM, n, m);
    n0 = n * (DUAL ? 128 : BN);
    m0 = tile.y + m * BM;
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
    ssrc[i] = a.Xs + m * a.xs_row;
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
  const int xo = wm * 2048, wo = (BM + wn * 16 * NF) * 128, so = (BM + BN) * 128 + (wm * 16 + (lane & 15)) * 4;
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
      const i8v xf = frag(buf + xo + 2048 * WM * m);
      const float xs = *reinterpret_cast<const float *>(buf + so + 64 * WM * m);
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

  if constexpr (DUAL) __syncthreads();  // (the first bytes of LDS hold maxima now)
  fp8_store<MF, NF, WM, WN, MODE>(a, acc, m0, m_end, n0, reinterpret_cast<uint32_t *>(smem));
}

// ---- the same tiles as a persistent pipeline -----------------------------------------------------
//
// For at least ST blocks of K. What the plain form above loses, per step of a 256 x 256
// tile (its matrix instructions take 0.85 us at the clock that they run at on real data): all waves read LDS at once behind the
// barrier, then multiply; the address of each load is 64-bit arithmetic on the vector unit; a tile's last stores and the next
// one's first loads overlap with nothing.
//   - The barrier of a step stands before its last two fragments of X: by then the wave holds all that it reads of this
//     stage, so behind it the next stage's first fragments are read, and the stage just left is filled again, under the
//     matrix instructions of those two. A fragment of W is read for the next step once its last product has been issued.
//   - The fma of a block product come a group later than its instruction (t, tb), in an order that scheduling barriers hold.
//   - A workgroup takes tile after tile; the stages of the next one are on their way before the last step of this one.
//   - Loads through buffer descriptors: one 32-bit offset a lane for all tiles, rows past the end and what lies behind a short
//     last block come back as zeros.

typedef uint32_t srd_t __attribute__((ext_vector_type(4)));

// 16 bytes a lane from buffer r to LDS: lane L's to byte address lds + 16 L. _if: only with `on` all ones (else 0), without a branch.
__device__ __forceinline__ void srd_dma16(const srd_t &r, uint32_t voff, uint32_t soff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds" ::"v"(voff), "s"(r), "s"(soff), "s"(lds)
               : "memory", "m0");
}
__device__ __forceinline__ void srd_dma16_if(const srd_t &r, uint32_t voff, uint32_t soff, uint32_t lds, uint32_t on) {
  asm volatile("s_mov_b32 m0, %3\n\ts_mov_b32 exec_lo, %4\n\ts_mov_b32 exec_hi, %4\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds\n\t"
               "s_mov_b64 exec, -1" ::"v"(voff), "s"(r), "s"(soff), "s"(lds), "s"(on)
               : "memory", "m0");
}

template <int MF, int NF, int WM, int WN, int ST, int MODE, bool HALF, bool TAIL = false>
__global__ void __launch_bounds__(64 * WM * WN) k_fp8_pipe(const Fp8MmArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int BM = 16 * MF * WM, BN = 16 * NF * WN, NW = WM * WN;
  constexpr int STAGE = (BM + BN) * 128, SCALES = ST * STAGE, SQ = 16 * BM;  // bytes: of a stage, before the scales, of four steps' scales
  constexpr int RL = (BM + BN) / 8, PER = RL / NW, XPER = BM / 8 / NW;  // loads of 8 rows: to a stage, to a wave, of them of X
  constexpr bool DUAL = MODE == FP8_GATE_UP, GATHER = MODE == FP8_GATE_UP;
  constexpr bool ONE = HALF || MODE != FP8_DENSE;  // a fragment of X at a time, or (dense, e4m3) the last two at once
  static_assert(!TAIL || MODE == FP8_DENSE, "short blocks");
  static_assert(MF >= 4 && MF % 2 == 0 && (!ONE || MF == 4) && RL % NW == 0 && BM / 8 % NW == 0 && BM / 64 <= NW, "tile");
  static_assert(!DUAL || (BN == 256 && NF % 2 == 0), "a tile of gate and up holds one block of 128 columns of each");
  static_assert(DUAL || 128 % (16 * NF) == 0, "a wave's rows of W lie in one block");
  static_assert(ST <= 4 && PER * (ST - 1) <= 63, "loads that vmcnt can count");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int wm = wave / WN, wn = wave % WN;
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char *)smem));
  const int nk = a.KB;
  const int units = MODE == FP8_DENSE ? a.units : __builtin_amdgcn_readfirstlane(*a.ntiles) * a.n_tiles;

  struct Buf {  // a buffer's address and size: descriptor words
    uint32_t lo, hi, bytes;
  };
  struct Tile {  // where the loads of a tile come from (wave-uniform, but for the gathered rows' offsets)
    Buf x, w, w2, s;
    uint32_t xoff[GATHER ? XPER : 1], soff;
    int last;  // TAIL: the step whose block is short
  };
  auto buf_of = [](const void *p, int64_t bytes) {
    const uint64_t q = reinterpret_cast<uint64_t>(p);
    return Buf{static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(q))),
               static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(q >> 32) & 0xffffu)),
               static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(bytes)))};
  };
  auto srd_of = [](const Buf &b) {
    return srd_t{static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(b.lo)), static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(b.hi)),
                 static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(b.bytes)), 0x00027000u};
  };
  // the tile to compute: rows m0 .. m_end, columns n0 .., scales of this wave's rows of W
  struct Place {
    int m0, m_end, n0, nk, split;  // (blocks of K of this unit)
    const float *ws, *ws2;
  };
  uint32_t off[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int j = wave + NW * i, c = (lane & 7) ^ (lane >> 3);
    int r = 8 * j + (lane >> 3);
    if (i >= XPER) {
      r -= BM;
      if constexpr (DUAL) r = 8 * NF * (r / (16 * NF)) + r % (8 * NF);  // row of gate (or up) behind n0
    }
    off[i] = static_cast<uint32_t>(r) * static_cast<uint32_t>(a.K) + 16 * c;
  }
  const uint32_t s_on = __builtin_amdgcn_readfirstlane(wave < BM / 64 ? ~0u : 0u);  // waves that load scales: 64 rows each
  // unit u: splits of K outermost; dense tiles in groups of 8 tiles of rows, columns by columns; experts' tiles:
  // fp8_expert_unit
  auto tile_at = [&](int u, Tile &f) {
    Place t;
    const uint8_t *W = a.W, *W2 = a.W2;
    const float *Ws = a.Ws, *W2s = a.W2s;
    int n;
    int k0 = 0;
    t.nk = nk;
    t.split = 0;
    if constexpr (MODE == FP8_DENSE) {
      const int tiles = a.m_tiles * a.n_tiles;
      if (a.splits > 1) {
        t.split = u / tiles;
        u -= t.split * tiles;
        k0 = static_cast<int>(static_cast<int64_t>(t.split) * nk / a.splits);
        t.nk = static_cast<int>(static_cast<int64_t>(t.split + 1) * nk / a.splits) - k0;
      }
      const int per = 8 * a.n_tiles, g = u / per, r = u - g * per, gm = min(8, a.m_tiles - 8 * g);
      n = r / gm;
      t.m0 = (8 * g + r - n * gm) * BM;
      t.m_end = a.M;
    } else {
      int m;
      const int4 q = fp8_expert_unit(a, u, BM, n, m);
      n = __builtin_amdgcn_readfirstlane(n);
      const int x = __builtin_amdgcn_readfirstlane(q.x);
      t.m0 = __builtin_amdgcn_readfirstlane(q.y + m * BM);
      t.m_end = __builtin_amdgcn_readfirstlane(q.z);
      if (x < 0) {
        W = a.Ss;
        W2 = a.S2;
        Ws = a.Sss;
        W2s = a.S2s;
      } else {
        W += x * a.w_stride;
        Ws += x * a.ws_stride;
        if constexpr (DUAL) {
          W2 += x * a.w_stride;
          W2s += x * a.ws_stride;
        }
      }
    }
    t.n0 = n * (DUAL ? 128 : BN);
    const int rows = min(BM, t.m_end - t.m0), cols = min(DUAL ? 128 : BN, a.N - t.n0);
    f.last = TAIL ? nk - 1 - k0 : 0;
    f.w = buf_of(W + static_cast<int64_t>(t.n0) * a.K + 128 * k0, static_cast<int64_t>(cols) * a.K - 128 * k0);
    if constexpr (DUAL) f.w2 = buf_of(W2 + static_cast<int64_t>(t.n0) * a.K, static_cast<int64_t>(cols) * a.K);
    const int nb = (DUAL ? t.n0 : min(t.n0 + 16 * NF * wn, a.N - 1)) >> 7;
    t.ws = Ws + static_cast<int64_t>(nb) * nk + k0;
    t.ws2 = DUAL ? W2s + static_cast<int64_t>(nb) * nk : nullptr;
    const int sr = wave * 64 + lane;  // row of this lane's scale (waves past the last do not load it)
    if constexpr (GATHER) {
      f.x = buf_of(a.X, a.x_rows * a.K);
      f.s = buf_of(a.Xs, a.x_rows * nk * 4);
#pragma unroll
      for (int i = 0; i < XPER; ++i) {
        const int r = 8 * (wave + NW * i) + (lane >> 3);
        f.xoff[i] = static_cast<uint32_t>(a.row_map[t.m0 + min(r, rows - 1)]) * static_cast<uint32_t>(a.K) + 16 * ((lane & 7) ^ (lane >> 3));
      }
      f.soff = static_cast<uint32_t>(a.row_map[t.m0 + min(sr, rows - 1)]) * static_cast<uint32_t>(a.xs_row * 4);
    } else {
      f.x = buf_of(a.X + static_cast<int64_t>(t.m0) * a.K + 128 * k0, static_cast<int64_t>(rows) * a.K - 128 * k0);
      f.s = buf_of(a.Xs + t.m0 * a.xs_row + k0, 4 * ((rows - 1) * a.xs_row + nk - k0));
      f.soff = static_cast<uint32_t>(sr) * static_cast<uint32_t>(a.xs_row * 4);
    }
    return t;
  };
  // load i of stage k of a tile, into the stage at LDS byte l
  // (chunks behind the end of a short block: offsets past the buffer, which read as zeros)
  const uint32_t behind = TAIL && 16 * ((lane & 7) ^ (lane >> 3)) >= (a.K & 127) ? 0x80000000u : 0u;
  auto issue1 = [&](const Tile &t, int k, uint32_t l, int i) {
    const int j = wave + NW * i;
    const uint32_t at = TAIL ? off[i] + (k == t.last ? behind : 0u) : off[i];
    if (i < XPER) {  // (known where the loop over i is unrolled: no branch)
      srd_dma16(srd_of(t.x), GATHER ? t.xoff[i < XPER ? i : 0] : at, 128 * k, l + 1024 * j);
    } else if constexpr (DUAL) {
      const bool up = (8 * j - BM) % (16 * NF) >= 8 * NF;
      srd_dma16(srd_of(Buf{up ? t.w2.lo : t.w.lo, up ? t.w2.hi : t.w.hi, t.w.bytes}), at, 128 * k, l + 1024 * j);
    } else {
      srd_dma16(srd_of(t.w), at, 128 * k, l + 1024 * j);
    }
  };
  // the scales of steps k .. k + 3 of a tile, at every fourth step: 16 bytes a row (single ones cost an address cycle a row and
  // step), into the next of four places; what lies behind a tile's last step is not used
  uint32_t place = 0;
  auto issue_s = [&](const Tile &t, int k) {
    const uint32_t on = (k & 3) == 0 ? s_on : 0u;
    srd_dma16_if(srd_of(t.s), t.soff, static_cast<uint32_t>(4 * k), lds0 + SCALES + place * SQ + wave * 1024,
                 __builtin_amdgcn_readfirstlane(on));
    place = (place + ((k & 3) == 0 ? 1 : 0)) & 3;
  };
  const int lo = (lane & 15) * 128 + (((lane >> 4) ^ (lane & 7)) * 16);
  const int xo = wm * 2048, wo = (BM + wn * 16 * NF) * 128, so = SCALES + (wm * 16 + (lane & 15)) * 16;
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
  auto x_of = [&](const char *p, int m) { return frag(p + xo + 2048 * WM * m); };
  auto scale_of = [&](uint32_t at, int m) { return *reinterpret_cast<const float *>(smem + at + so + 256 * WM * m); };
  auto add = [&](f4 &c, const f4 &v, float s) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = fmaf(v[i], s, c[i]);
  };
  auto hold = [] { __builtin_amdgcn_sched_barrier(0); };
  auto barrier = [&] {
    hold();
    __builtin_amdgcn_s_barrier();
    hold();
    asm volatile("" ::: "memory");
  };

  const int G = gridDim.x;
  int u = blockIdx.x;
  if (G % 8 == 0) u = (u & 7) * (G >> 3) + (u >> 3);  // workgroups are dealt to the 8 XCDs in turn
  if (u >= units) return;
  Tile from;
  Place at = tile_at(u, from);
#pragma unroll
  for (int s = 0; s < ST; ++s) {
#pragma unroll
    for (int i = 0; i < PER; ++i) issue1(from, s, lds0 + s * STAGE, i);
    issue_s(from, s);
  }
  wait_loads<PER *(ST - 1)>();
  barrier();
  i8v wf[NF], xf[4];
  float xs[4];
#pragma unroll
  for (int n = 0; n < NF; ++n) wf[n] = frag(smem + wo + 2048 * n);
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    xf[m] = x_of(smem, m);
    xs[m] = scale_of(0, m);
  }
  // HALF: the converted fragments, all of W (made at a step's start) and one of X (made ahead)
  h8 wh[HALF ? NF : 1][4], xh[4];
  if constexpr (HALF)
#pragma unroll
    for (int j = 0; j < 4; ++j) xh[j] = fp8_to_h8(xf[0][2 * j], xf[0][2 * j + 1]);
  uint32_t sb = 0, cb = 0;  // byte offsets of the current stage and of its scales among them
  for (; u < units; u += G) {
    f4 acc[NF][MF], t[NF], tb = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < NF; ++n) {
      t[n] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int m = 0; m < MF; ++m) acc[n][m] = f4{0.f, 0.f, 0.f, 0.f};
    }
    struct Sc {
      float g, u;
    };
    auto of = [](const Sc &s, int n) { return DUAL && n >= NF / 2 ? s.u : s.g; };
    Sc sp = {0.f, 0.f}, sq = {0.f, 0.f};  // of the products that wait in t[NF - 1] and tb
    Tile next = from;  // (behind the last tile: loads that nothing reads)
    Place then = at;
    if (u + G < units) then = tile_at(u + G, next);
    const float *ws = at.ws, *ws2 = at.ws2;
    float w0 = uniform_load(ws, 0), w1 = DUAL ? uniform_load(ws2, 0) : 0.f;
    const int nk = at.nk;
    // step k with the first MA of MF fragments of X (all, or 2)
    auto step = [&](auto ma, int k) {
      constexpr int MA = decltype(ma)::value;
      const uint32_t sn = sb + STAGE == ST * STAGE ? 0 : sb + STAGE;
      const char *buf = smem + sb, *nbuf = smem + sn;
      const uint32_t cn = k + 1 == nk || (k & 3) == 3 ? (((cb / SQ) + 1) & 3) * SQ : cb + 4;
      const int kn = k + 1 < nk ? k + 1 : k;
      const float w0n = uniform_load(ws, kn), w1n = DUAL ? uniform_load(ws2, kn) : 0.f;
      auto scales = [&](int m) { return Sc{xs[m & 3] * w0, DUAL ? xs[m & 3] * w1 : 0.f}; };
      // the stage to load: ST steps on, from the next tile once this one's are all on their way
      const int kk = k + ST < nk ? k + ST : k + ST - nk;
      auto turn = [&] {
        const bool now = k + ST == nk;
        auto pick = [&](Buf &b, const Buf &n) {
          b.lo = now ? n.lo : b.lo;
          b.hi = now ? n.hi : b.hi;
          b.bytes = now ? n.bytes : b.bytes;
        };
        pick(from.w, next.w);
        if constexpr (DUAL) {
          from.w2.lo = now ? next.w2.lo : from.w2.lo;
          from.w2.hi = now ? next.w2.hi : from.w2.hi;
        }
        if constexpr (GATHER) {
#pragma unroll
          for (int i = 0; i < XPER; ++i) from.xoff[i] = now ? next.xoff[i] : from.xoff[i];
          from.soff = now ? next.soff : from.soff;
        } else {
          pick(from.x, next.x);
          pick(from.s, next.s);
          if constexpr (TAIL) from.last = now ? next.last : from.last;
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this wave has read all of the stage
        wait_loads<PER *(ST - 2)>();  // its loads of the next one have arrived (its load of scales, which some waves lack, not counted)
        barrier();
      };
      if constexpr (ONE) {
        // Fragment by fragment: while the matrix instructions of one run, the last one's products are added and (HALF: 16 cycles
        // each, 4 to issue) the next one is converted, three vector instructions to each of them. Fragment m + 2, or the next
        // step's, is read meanwhile; the barrier stands before the last two.
        i8v xr[MA + 2];
        float xv[MA + 2];
        xr[0] = xf[0];
        xr[1] = xf[1];
        xv[0] = xs[0];
        xv[1] = xs[1];
#pragma unroll
        for (int m = 0; m < MA; ++m) {
          if (m == MA - 2) turn();
          xr[m + 2] = m + 2 < MA ? x_of(buf, m + 2) : x_of(nbuf, m + 2 - MA);
          xv[m + 2] = m + 2 < MA ? scale_of(cb, m + 2) : scale_of(cn, m + 2 - MA);
          if (HALF && m == 0)
#pragma unroll
            for (int n = 0; n < NF; ++n)
#pragma unroll
              for (int j = 0; j < 4; ++j) wh[HALF ? n : 0][j] = fp8_to_h8(wf[n][2 * j], wf[n][2 * j + 1]);
          const Sc s = {xv[m] * w0, DUAL ? xv[m] * w1 : 0.f};
          // the loads of the stage ST steps on, spread over what is left of the step: issued together they hold up the instructions
          // behind them until the address unit has taken them all
          constexpr int SUB = HALF ? 1 : NF, BY = NF / SUB;  // parts of a fragment's products, columns to a part
          constexpr int SLOTS = 2 * SUB;
          h8 xn[HALF ? 4 : 1];
#pragma unroll
          for (int p = 0; p < SUB; ++p) {
#pragma unroll
            for (int n = p * BY; n < (p + 1) * BY; ++n) {
              add(acc[n][(m + MA - 1) % MA], t[n], of(sp, n));
              t[n] = f4{0.f, 0.f, 0.f, 0.f};
              if constexpr (!HALF) t[n] = fp8_block<false>(wf[n], xr[m]);
            }
            if constexpr (HALF) {
#pragma unroll
              for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int n = p * BY; n < (p + 1) * BY; ++n) t[n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wh[HALF ? n : 0][j], xh[j], t[n], 0, 0, 0);
              if (p == SUB - 1)
#pragma unroll
                for (int j = 0; j < 4; ++j) xn[HALF ? j : 0] = fp8_to_h8(xr[m + 1][2 * j], xr[m + 1][2 * j + 1]);
#pragma unroll
              for (int i = 0; i < 4 * BY; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // a matrix instruction
                __builtin_amdgcn_sched_group_barrier(0x002, 3, 0);  // three vector instructions
              }
            }
            if (m == MA - 1)
#pragma unroll
              for (int n = p * BY; n < (p + 1) * BY; ++n) wf[n] = frag(nbuf + wo + 2048 * n);
            hold();
            if (m >= MA - 2) {
              const int q = (m - (MA - 2)) * SUB + p;
#pragma unroll
              for (int i = q * PER / SLOTS; i < (q + 1) * PER / SLOTS; ++i) issue1(from, kk, lds0 + sb, i);
              if (q == SLOTS - 1) issue_s(from, kk);
              hold();
            }
          }
          if constexpr (HALF)
#pragma unroll
            for (int j = 0; j < 4; ++j) xh[j] = xn[j];
          sp = s;
        }
        xf[0] = xr[MA];
        xf[1] = xr[MA + 1];
        xs[0] = xv[MA];
        xs[1] = xv[MA + 1];
      } else {
        Sc sc = {0.f, 0.f};
#pragma unroll
        for (int m = 0; m < MF - 2; ++m) {
          xf[(m + 2) & 3] = x_of(buf, m + 2);
          xs[(m + 2) & 3] = scale_of(cb, m + 2);
          const Sc s = scales(m);
#pragma unroll
          for (int n = 0; n < NF; ++n) {
            if (m > 0) {
              add(acc[n][m - 1], t[n], of(sc, n));
            } else if (n == 0) {
              add(acc[NF - 1][MF - 2], t[NF - 1], of(sp, NF - 1));
              add(acc[NF - 1][MF - 1], tb, of(sq, NF - 1));
            }
            t[n] = fp8_block<false>(wf[n], xf[m & 3]);
            hold();
          }
          sc = s;
        }
        const Sc s6 = scales(MF - 2), s7 = scales(MF - 1);
        turn();
#pragma unroll
        for (int n = 0; n < NF; ++n) {
          if (n == 0) {
            xf[MF & 3] = x_of(nbuf, 0);
            xs[MF & 3] = scale_of(cn, 0);
          }
          if (n == 1) {
            xf[(MF + 1) & 3] = x_of(nbuf, 1);
            xs[(MF + 1) & 3] = scale_of(cn, 1);
          }
          add(acc[n][MF - 3], t[n], of(sc, n));
          if (n > 0) {
            add(acc[n - 1][MF - 2], t[n - 1], of(s6, n - 1));
            add(acc[n - 1][MF - 1], tb, of(s7, n - 1));
          }
          t[n] = fp8_block<false>(wf[n], xf[(MF - 2) & 3]);
          tb = fp8_block<false>(wf[n], xf[(MF - 1) & 3]);
          wf[n] = frag(nbuf + wo + 2048 * n);
#pragma unroll
          for (int i = n * PER / NF; i < (n + 1) * PER / NF; ++i) issue1(from, kk, lds0 + sb, i);
          if (n == NF - 1) issue_s(from, kk);
          hold();
        }
        if constexpr (MF % 4 != 0) {  // the ring's first places are fragments 0 and 1
          const i8v x0 = xf[MF & 3], x1 = xf[(MF + 1) & 3];
          const float f0 = xs[MF & 3], f1 = xs[(MF + 1) & 3];
          xf[0] = x0;
          xf[1] = x1;
          xs[0] = f0;
          xs[1] = f1;
        }
        sp = s6;
        sq = s7;
      }
      w0 = w0n;
      w1 = w1n;
      sb = sn;
      cb = cn;
    };
    auto steps = [&](auto ma) {
      for (int k = 0; k < nk; ++k) step(ma, k);
      if constexpr (ONE)
#pragma unroll
        for (int n = 0; n < NF; ++n) add(acc[n][decltype(ma)::value - 1], t[n], of(sp, n));
    };
    if constexpr (MODE != FP8_DENSE) {  // experts' tiles are often not full: no instructions for fragments that no row is in
      const int rows = __builtin_amdgcn_readfirstlane(at.m_end - at.m0);
      if (rows > 2 * 16 * WM) steps(std::integral_constant<int, 4>{});
      else steps(std::integral_constant<int, 2>{});
    } else {
      steps(std::integral_constant<int, MF>{});
    }
    if constexpr (!ONE) {
      add(acc[NF - 1][MF - 2], t[NF - 1], of(sp, NF - 1));
      add(acc[NF - 1][MF - 1], tb, of(sq, NF - 1));
    }
    fp8_store<MF, NF, WM, WN, MODE>(a, acc, at.m0, at.m_end, at.n0, reinterpret_cast<uint32_t *>(smem + SCALES + 4 * SQ), at.split);
    at = then;
  }
  wait_loads<0>();  // (nothing may arrive in LDS that is another workgroup's)
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

// The pipeline: as many workgroups as the device holds at once, at most `units`.
template <int MF, int NF, int WM, int WN, int ST, int MODE, bool HALF, bool TAIL = false>
int fp8_pipe_launch(const Fp8MmArgs &a, int64_t units, hipStream_t s) {
  constexpr int BM = 16 * MF * WM, BN = 16 * NF * WN;
  constexpr int LDS = ST * (BM + BN) * 128 + 64 * BM + (MODE == FP8_GATE_UP ? 4 * WN * BM : 0);
  static_assert(LDS <= 160 * 1024, "LDS");
  static std::atomic<uint64_t> raised{0};
  static std::atomic<int64_t> resident[64];
  auto *fn = &k_fp8_pipe<MF, NF, WM, WN, ST, MODE, HALF, TAIL>;
  int rc = ensure_lds_limit(reinterpret_cast<const void *>(fn), LDS, raised, "fp8 product"), per_cu = 1;
  if (!rc) rc = resident_per_cu(reinterpret_cast<const void *>(fn), 64 * WM * WN, LDS, resident, per_cu, "fp8 product");
  if (rc) return rc;
  const int64_t most = static_cast<int64_t>(device_cu_count()) * per_cu;
  hipLaunchKernelGGL(fn, dim3(static_cast<unsigned>(units < most ? units : most)), dim3(64 * WM * WN), LDS, s, a);
  return check_launch("fp8 product");
}

}  // namespace vybdq
