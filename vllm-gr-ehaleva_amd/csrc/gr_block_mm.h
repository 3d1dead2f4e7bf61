// Matrix product tile shared by the 8-bit block-scaled projections
// (gr_block_fp8.hip) and the experts' layers (gr_experts.hip).
//
//   y[t, n] = sum_k x[t, k] w[n, k]                       (fp16, bf16)
//   y[t, n] = sum_b xs[t, b] ws[n / 128, b] sum_{k in b} x[t, k] w[n, k]   (e4m3)
//
// A stage is 128 bytes of each row of both operands -- 64 features of 16 bits, or
// one block of 128 e4m3 features -- and lies in LDS as rows of 128 bytes whose
// 16-byte chunks are XOR-swizzled by the row, moved there straight from global
// memory, ST stages in flight.  Lane l of a fragment of 16 rows reads chunks
// l / 16 and 4 + l / 16 of row l % 16: the two 32-deep operands of the 16-bit
// instructions, or the one 128-deep operand of the 8-bit one (which features of
// the stage sit where does not matter as long as both operands agree).  The
// weights are the A operand, so a lane holds four neighbouring columns of one row
// t of the result and needs that row's scale alone.  A block's 128 products are
// summed by the matrix core into a zeroed accumulator, scaled and added in float32.
//
// The 8-bit matrix instruction adds products in groups of 8, each cut off (towards
// zero) below 2^-13 of the group's largest product's power of two: about 1.5e-5 of
// a result of ordinary operands, measured.  A 16-bit result (2^-9 and 2^-12 of
// rounding) does not show that.  A float32 one would, and so would one that is
// rounded to e4m3 again, where values at a border move by a whole step: those are
// EXACT, with the e4m3 operands converted to fp16 (which holds each of them) ahead
// of the 16-bit instruction, at half its rate, and all sums in float32.
#pragma once

#include "gr_experts.h"
#include "gr_mfma_tile.h"

namespace gr {
namespace {

typedef float mm4_t __attribute__((__vector_size__(16)));
typedef int mm4i_t __attribute__((__vector_size__(16)));
typedef int mm8i_t __attribute__((__vector_size__(32)));

enum { MM_PLAIN = 0, MM_SWIGLU = 1, MM_SWIGLU_Q = 2, MM_PLAIN_Q = 3 };

struct MmArgs {
  const uint8_t* x;
  int64_t x_stride;  // bytes
  const float* xs;   // e4m3: row scales
  int64_t xs_row, xs_grp;
  const uint8_t* w;
  int64_t w_stride;  // bytes
  const float* ws;   // e4m3: block scales, groups contiguous
  void* out;
  int64_t out_stride;  // elements
  float* out_scale;    // *_Q
  int64_t os_row, os_grp;
  int M, N;    // rows, output columns (SwiGLU: 2 N weight rows)
  int kbytes;  // bytes of a row, a multiple of 16
  int out_type;
  int tiles_m, tiles_n;
  // experts: row tiles {expert, first row, rows} of the rows sorted by expert
  const int4* tiles;
  const int* num_tiles;
  const int* slot;  // token * top_k + choice of each sorted row
  int gather;       // x row of sorted row p: slot[p] / gather; 0: p
  int scatter;      // output row: slot[p]; 0: p
  int64_t w_expert, ws_expert;  // bytes, elements
};

// The e4m3 number nearest to x / s, as a float32 that rounds to it: the quotient
// to within an ulp, moved off a border between two e4m3 numbers (where its last
// bit is 0) to the side that the exact remainder says.  r = 1 / s.  Below 2^-11
// everything rounds to 0.
__device__ inline float quant_div(float x, float s, float r) {
  float q = x * r;
  q = fmaf(fmaf(-q, s, x), r, q);
  const float rem = fmaf(-q, s, x);
  const uint32_t b = __builtin_bit_cast(uint32_t, q);
  if (fabsf(q) >= 0x1p-11f && rem != 0.f && (b & 1) == 0) {
    const bool up = ((__builtin_bit_cast(uint32_t, rem) ^ b) >> 31) == 0;  // |exact| > |q|
    q = __builtin_bit_cast(float, up ? b + 1 : b - 1);
  }
  return q;
}
// scale of a group from the bits of its largest |x| (a NaN's are the largest)
__device__ inline float quant_scale(uint32_t amax_bits) {
  const float t = __builtin_bit_cast(float, amax_bits) / 448.0f;
  return t < 0x1p-80f ? 0x1p-80f : t;
}
__device__ inline uint32_t quant_pack4(const float (&v)[4], float s, float r) {
  int p = 0;
  p = __builtin_amdgcn_cvt_pk_fp8_f32(quant_div(v[0], s, r), quant_div(v[1], s, r), p, false);
  p = __builtin_amdgcn_cvt_pk_fp8_f32(quant_div(v[2], s, r), quant_div(v[3], s, r), p, true);
  return (uint32_t)p;
}

template <int DT> __device__ inline mm4_t mm_mma(u32x4_t a, u32x4_t b, mm4_t c) {
  if constexpr (DT == GR_DTYPE_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                   0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0,
                                                  0, 0);
}

// cnt neighbouring results in the output's type; vec: all four, aligned
__device__ inline void mm_store(void* out, int type, int64_t at, const float (&v)[4], int cnt, bool vec) {
  if (type == GR_DTYPE_F32) {
    float* o = static_cast<float*>(out) + at;
    if (vec) *reinterpret_cast<mm4_t*>(o) = mm4_t{v[0], v[1], v[2], v[3]};
    else
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (u < cnt) o[u] = v[u];
    return;
  }
  const bool bf = type == GR_DTYPE_BF16;
  const uint32_t lo = bf ? Mma<GR_DTYPE_BF16>::pack2(v[0], v[1]) : Mma<GR_DTYPE_F16>::pack2(v[0], v[1]);
  const uint32_t hi = bf ? Mma<GR_DTYPE_BF16>::pack2(v[2], v[3]) : Mma<GR_DTYPE_F16>::pack2(v[2], v[3]);
  uint16_t* o = static_cast<uint16_t*>(out) + at;
  if (vec) {
    *reinterpret_cast<u32x2_t*>(o) = u32x2_t{lo, hi};
    return;
  }
  const uint32_t p[2] = {lo, hi};
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (u < cnt) o[u] = (uint16_t)(p[u >> 1] >> (16 * (u & 1)));
}

// One dword per lane from global memory into LDS: lane i's lands at lds + 4 i.
__device__ inline void dma_v1(uint32_t lds, const void* addr) {
  const uint32_t m = __builtin_amdgcn_readfirstlane(lds);
  uint32_t save;
  __asm__ volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %2, off\n\ts_mov_b32 m0, %0"
                   : "=&s"(save) : "s"(m), "v"(addr) : "memory");
}

template <int N> __device__ __forceinline__ void mm_wait_barrier() {
  __asm__ volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// The workgroup's tile: row tiles go in groups of G, within a group the column
// tiles one after the other (their weights are shared by the group's row tiles,
// its rows by all of them), and the sequence is cut into one run per XCD, so that
// what neighbours share is read into one L2.
__device__ inline bool mm_tile(const MmArgs& a, int tiles_m, int& mt, int& nt) {
  constexpr int G = 8;
  const int total = tiles_m * a.tiles_n;
  const int per = (total + 7) >> 3;
  const int local = blockIdx.x >> 3, xcd = blockIdx.x & 7;
  const int p = xcd * per + local;
  if (local >= per || p >= total) return false;
  const int group = p / (G * a.tiles_n), in = p - group * G * a.tiles_n;
  const int rows = min(G, tiles_m - group * G);
  nt = in / rows;
  mt = group * G + in - nt * rows;
  return true;
}

// XT: element type of both operands.  WM x WN waves over a BM x BN tile (BN weight
// rows; with SwiGLU 16 gate rows and the 16 up rows of the same columns alternate).
template <int XT, int BM, int BN, int WM, int WN, int ST, int MODE, bool EXPERTS, bool EXACT>
__global__ __launch_bounds__(64 * WM * WN) void block_mm(MmArgs a) {
  constexpr bool F8 = XT == GR_DTYPE_FP8_E4M3;
  static_assert(F8 || !EXACT, "16-bit sums are exact as they are");
  constexpr bool GATED = MODE == MM_SWIGLU || MODE == MM_SWIGLU_Q;
  constexpr bool QUANT = MODE == MM_SWIGLU_Q || MODE == MM_PLAIN_Q;
  constexpr int NW = WM * WN;
  constexpr int TILE = (BM + BN) * 128;                 // bytes of a stage
  constexpr int STAGE = TILE + (F8 ? NW * 256 : 0);     // and the row scales
  constexpr int LPS = (BM + BN) / 8 / NW;               // transfers per wave and stage, 8 rows each
  constexpr int OPS = LPS + (F8 ? 1 : 0);
  constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
  constexpr int OC = GATED ? BN / 2 : BN;               // output columns of the tile
  static_assert((BM + BN) % (8 * NW) == 0 && BM <= NW * 64, "whole transfers");
  static_assert(BM % (16 * WM) == 0 && BN % (16 * WN) == 0 && (!GATED || FN % 2 == 0), "whole fragments");
  static_assert(OC / WN <= 128 && 128 % (OC / WN) == 0, "a wave's columns share a weight block");
  static_assert(!QUANT || OC == 128, "a tile's columns are one group of the result");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[ST * STAGE];

  const int tiles_m = EXPERTS ? __builtin_amdgcn_readfirstlane(*a.num_tiles) : a.tiles_m;
  int mt, nt;
  if (!mm_tile(a, tiles_m, mt, nt)) return;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  int m0 = mt * BM, m_end = a.M;
  const uint8_t* w = a.w;
  const float* ws = a.ws;
  if constexpr (EXPERTS) {
    const int4 t = a.tiles[mt];
    const int e = __builtin_amdgcn_readfirstlane(t.x);
    m0 = __builtin_amdgcn_readfirstlane(t.y);
    m_end = m0 + __builtin_amdgcn_readfirstlane(t.z);
    w += e * a.w_expert;
    if constexpr (F8) ws += e * a.ws_expert;
  }
  const int n0 = nt * OC;

  // Transfer i of a stage moves LDS rows 8 (wave + NW i) .. + 7 (x rows, then w
  // rows); lane l lands on row l >> 3, chunk l & 7 of them and fetches the logical
  // chunk (l & 7) ^ (row & 7).  Rows past the tile's last repeat it (their results
  // are not stored).
  const int ch = ((lane & 7) ^ (lane >> 3)) * 16;
  auto x_row = [&](int r) -> int64_t {
    const int p = min(m0 + r, m_end - 1);
    if constexpr (EXPERTS) return a.gather ? a.slot[p] / a.gather : p;
    else return p;
  };
  const uint8_t* src[LPS];
#pragma unroll
  for (int i = 0; i < LPS; ++i) {
    const int row = 8 * (wave + NW * i) + (lane >> 3);
    if (row < BM) {
      src[i] = a.x + x_row(row) * a.x_stride + ch;
    } else {
      const int b = row - BM;
      const int64_t n = GATED ? min(n0 + (b >> 5) * 16 + (b & 15), a.N - 1) + (int64_t)((b >> 4) & 1) * a.N
                              : min(n0 + b, a.N - 1);
      src[i] = w + n * a.w_stride + ch;
    }
  }
  const float* xsrc = F8 ? a.xs + x_row(min(wave * 64 + lane, BM - 1)) * a.xs_row : nullptr;
  const uint32_t lds0 = (uint32_t)reinterpret_cast<uintptr_t>(lds);
  const int n = (a.kbytes + 127) >> 7;
  auto fetch = [&](int s, int buf) __attribute__((always_inline)) {
    const bool part = (s + 1) * 128 > a.kbytes;  // a short last stage: zeros behind its end
#pragma unroll
    for (int i = 0; i < LPS; ++i) {
      const uint8_t* p = src[i] + (int64_t)s * 128;
      if (part && s * 128 + ch >= a.kbytes) p = reinterpret_cast<const uint8_t*>(g_zero16);
      dma_v(lds0 + (uint32_t)(buf * STAGE + (wave + NW * i) * 1024), p);
    }
    if constexpr (F8) dma_v1(lds0 + (uint32_t)(buf * STAGE + TILE + wave * 256), xsrc + s * a.xs_grp);
  };

  const int r16 = lane & 15, q = lane >> 4;
  const int fch[2] = {(q ^ (r16 & 7)) * 16, ((4 + q) ^ (r16 & 7)) * 16};
  const int xo = (wm * (BM / WM) + r16) * 128, wo = (BM + wn * (BN / WN) + r16) * 128;
  mm4_t acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j) acc[i][j] = mm4_t{0.f, 0.f, 0.f, 0.f};
  // scales of this wave's weight block(s): gate's and up's with SwiGLU
  const int kb = n, nb0 = (n0 + wn * (OC / WN)) >> 7;
  const int nb_last = ((a.N + 127) >> 7) - 1;
  const float* ws0 = F8 ? ws + (int64_t)min(nb0, nb_last) * kb : nullptr;
  const float* ws1 = F8 && GATED ? ws0 + (int64_t)(nb_last + 1) * kb : ws0;

  auto stage = [&](int s, int buf) __attribute__((always_inline)) {
    const uint8_t* p = lds + buf * STAGE;
    u32x4_t wf[2][FN];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < FN; ++i) wf[h][i] = *reinterpret_cast<const u32x4_t*>(p + wo + fch[h] + i * 2048);
    u32x4_t wh[EXACT ? 4 : 1][FN];  // as fp16
    if constexpr (EXACT)
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int z = 0; z < 4; ++z)
          wh[z][i] = Fp8Cvt<GR_DTYPE_F16>::x8(wf[z >> 1][i][2 * (z & 1)], wf[z >> 1][i][2 * (z & 1) + 1]);
    float s0 = 0.f, s1 = 0.f;
    if constexpr (F8) {
      s0 = ws0[s];
      if constexpr (GATED) s1 = ws1[s];
    }
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      const u32x4_t x0 = *reinterpret_cast<const u32x4_t*>(p + xo + fch[0] + j * 2048);
      const u32x4_t x1 = *reinterpret_cast<const u32x4_t*>(p + xo + fch[1] + j * 2048);
      if constexpr (F8) {
        const float xs = *reinterpret_cast<const float*>(p + TILE + (wm * (BM / WM) + j * 16 + r16) * 4);
        const float c0 = xs * s0, c1 = GATED ? xs * s1 : c0;
        if constexpr (EXACT) {
          const u32x4_t xh[4] = {Fp8Cvt<GR_DTYPE_F16>::x8(x0[0], x0[1]), Fp8Cvt<GR_DTYPE_F16>::x8(x0[2], x0[3]),
                                 Fp8Cvt<GR_DTYPE_F16>::x8(x1[0], x1[1]), Fp8Cvt<GR_DTYPE_F16>::x8(x1[2], x1[3])};
#pragma unroll
          for (int i = 0; i < FN; ++i) {
            mm4_t t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int z = 0; z < 4; ++z) t = mm_mma<GR_DTYPE_F16>(wh[z][i], xh[z], t);
            const float c = GATED && (i & 1) ? c1 : c0;
#pragma unroll
            for (int u = 0; u < 4; ++u) acc[i][j][u] = fmaf(t[u], c, acc[i][j][u]);
          }
          continue;
        }
        const mm8i_t xv = __builtin_shufflevector(__builtin_bit_cast(mm4i_t, x0), __builtin_bit_cast(mm4i_t, x1), 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
        for (int i = 0; i < FN; ++i) {
          const mm8i_t wv = __builtin_shufflevector(__builtin_bit_cast(mm4i_t, wf[0][i]), __builtin_bit_cast(mm4i_t, wf[1][i]), 0, 1, 2, 3, 4, 5, 6, 7);
          const mm4_t t = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv, xv, mm4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
          const float c = GATED && (i & 1) ? c1 : c0;
#pragma unroll
          for (int u = 0; u < 4; ++u) acc[i][j][u] = fmaf(t[u], c, acc[i][j][u]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < FN; ++i) acc[i][j] = mm_mma<XT>(wf[0][i], x0, acc[i][j]);
#pragma unroll
        for (int i = 0; i < FN; ++i) acc[i][j] = mm_mma<XT>(wf[1][i], x1, acc[i][j]);
      }
    }
  };

  // stage s has landed when all but the ST - 2 younger ones' transfers have; past
  // its barrier nobody reads stage s - 1, whose buffer takes stage s + ST - 1
#pragma unroll
  for (int s = 0; s < ST - 1; ++s)
    if (s < n) fetch(s, s);
  int buf = 0;
  for (int s = 0; s < n; ++s) {
    if (s + ST - 1 <= n) mm_wait_barrier<(ST - 2) * OPS>();
    else mm_wait_barrier<0>();
    if (s + ST - 1 < n) fetch(s + ST - 1, buf == 0 ? ST - 1 : buf - 1);
    stage(s, buf);
    buf = buf + 1 == ST ? 0 : buf + 1;
  }

  // fragment (i, j), register u: column 16 i + 4 (lane / 16) + u, row 16 j + lane % 16
  constexpr int STEP = GATED ? 2 : 1, FO = FN / STEP;  // output fragments
  auto value = [&](int i, int j, float (&v)[4]) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if constexpr (GATED) {
        const float g = acc[2 * i][j][u];
        v[u] = g / (1.0f + __expf(-g)) * acc[2 * i + 1][j][u];
      } else {
        v[u] = acc[i][j][u];
      }
    }
  };
  const int c0 = n0 + wn * (OC / WN) + 4 * q;
  auto out_row = [&](int r) -> int64_t {
    if constexpr (EXPERTS) return a.scatter ? a.slot[m0 + r] : m0 + r;
    else return m0 + r;
  };
  if constexpr (QUANT) {
    // the group's largest value: over the lane's columns, the four lanes of the
    // row, then the waves of the row through LDS
    uint32_t* part = reinterpret_cast<uint32_t*>(lds);  // [WN][BM]
    __syncthreads();
    float v[FO][FM][4];
    uint32_t am[FM];
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      am[j] = 0;
#pragma unroll
      for (int i = 0; i < FO; ++i) {
        value(i, j, v[i][j]);
        if (c0 + 16 * i < a.N)
#pragma unroll
          for (int u = 0; u < 4; ++u) am[j] = max(am[j], __builtin_bit_cast(uint32_t, v[i][j][u]) & 0x7FFFFFFFu);
      }
      am[j] = max(am[j], (uint32_t)__shfl_xor((int)am[j], 16, 64));
      am[j] = max(am[j], (uint32_t)__shfl_xor((int)am[j], 32, 64));
      if (q == 0) part[wn * BM + wm * (BM / WM) + j * 16 + r16] = am[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      const int r = wm * (BM / WM) + j * 16 + r16;
      uint32_t m = 0;
#pragma unroll
      for (int k = 0; k < WN; ++k) m = max(m, part[k * BM + r]);
      if (m0 + r >= m_end) continue;
      const float s = quant_scale(m), rs = 1.0f / s;
      const int64_t orow = out_row(r);
      if (wn == 0 && q == 0) a.out_scale[orow * a.os_row + nt * a.os_grp] = s;
      uint8_t* o = static_cast<uint8_t*>(a.out) + orow * a.out_stride;
#pragma unroll
      for (int i = 0; i < FO; ++i)
        if (c0 + 16 * i < a.N) *reinterpret_cast<uint32_t*>(o + c0 + 16 * i) = quant_pack4(v[i][j], s, rs);
    }
  } else {
    const bool vec = a.N % 4 == 0 && a.out_stride % 4 == 0;  // whole groups of four columns, each aligned
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      const int r = wm * (BM / WM) + j * 16 + r16;
      if (m0 + r >= m_end) continue;
      const int64_t o0 = out_row(r) * a.out_stride;
#pragma unroll
      for (int i = 0; i < FO; ++i) {
        const int col = c0 + 16 * i;
        if (col >= a.N) continue;
        float v[4];
        value(i, j, v);
        mm_store(a.out, a.out_type, o0 + col, v, vec ? 4 : min(4, a.N - col), vec);
      }
    }
  }
}

template <int XT, int BM, int BN, int WM, int WN, int ST, int MODE, bool EXPERTS, bool EXACT>
void launch_mm(MmArgs a, int tiles_m, hipStream_t stream) {
  constexpr int OC = MODE == MM_SWIGLU || MODE == MM_SWIGLU_Q ? BN / 2 : BN;
  a.tiles_m = tiles_m;
  a.tiles_n = (a.N + OC - 1) / OC;
  const int64_t total = (int64_t)tiles_m * a.tiles_n;
  hipLaunchKernelGGL((block_mm<XT, BM, BN, WM, WN, ST, MODE, EXPERTS, EXACT>), dim3((unsigned)((total + 7) / 8 * 8)),
                     dim3(64 * WM * WN), 0, stream, a);
}

}  // namespace
}  // namespace gr
