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
// a result of ordinary operands, measured.  A 16-bit result (2^-8 and 2^-11 of
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

// out_type of the experts' float32 results on their way to the sum over a token's
// experts: fp16 multiples of a power of two for each row's columns of one wave, so
// that the largest (of the finite ones) is within [2^14, 2^15): 2^-11 of a value that is
// not 2^28 times smaller than its neighbours.  Half the bytes of float32, which are most
// of what many tokens move (8192 tokens, 8 of 64 experts of 768: 770 us against 860).
constexpr int MM_OUT_SCALED = 16;

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
  int8_t* out_exp;     // MM_OUT_SCALED: log2 of the multiples' unit, [row][columns / a wave's]
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
// N values over their scale.  x r is within two ulps of x / s, so the side of a border
// is known unless x r lies within four of one: the borders of normal e4m3 numbers are
// where the 20 bits below their mantissa are one half.  Such values, and (low) any below
// the normal numbers but 0, are divided as above, which is rarely any wave's business.
template <int N> __device__ inline void quant_values(const float (&v)[N], float s, float r, bool low, float (&q)[N]) {
  uint32_t near = ~0u;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    q[i] = v[i] * r;
    near = min(near, (__builtin_bit_cast(uint32_t, q[i]) << 12) + 0x80004000u);
  }
  if (low || near < 0x8000u)
#pragma unroll
    for (int i = 0; i < N; ++i) q[i] = quant_div(v[i], s, r);
}
constexpr float QUANT_LOW = 0x1.0001p-6f;  // (a little over 2^-6, for the roundings)
// whether any value but 0 is below the normal e4m3 numbers (2^-6) of its scale
template <int N> __device__ inline bool quant_low(const float (&v)[N], float s) {
  uint32_t low = ~0u;
#pragma unroll
  for (int i = 0; i < N; ++i) low = min(low, (__builtin_bit_cast(uint32_t, v[i]) & 0x7FFFFFFFu) - 1u);
  return low != ~0u && __builtin_bit_cast(float, low + 1u) < s * QUANT_LOW;
}
// scale of a group from the bits of its largest |x| (a NaN's are the largest)
__device__ inline float quant_scale(uint32_t amax_bits) {
  const float t = __builtin_bit_cast(float, amax_bits) / 448.0f;
  return t < 0x1p-80f ? 0x1p-80f : t;
}
__device__ inline uint32_t fp8_pack4(const float* q) {
  const int p = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], p, true);
}

struct QuantArgs {
  uint8_t* out;
  int64_t out_stride;
  float* scale;
  int64_t scale_row, scale_grp;
  const void* x;
  int64_t x_stride;
  int T, K, groups;
};

// One group of 128 features per 8 lanes, 16 features a lane (wide loads and stores);
// a workgroup's groups are neighbours in their row.  Bound by memory: ROWS rows below
// each other keep that many pairs of loads on their way, and their scales, which lie side
// by side, reach one line together.
template <int DT, int ROWS> __device__ __forceinline__ void quant_group(const QuantArgs& a, uint32_t item, int l) {
  using E = Elem<DT>;
  using S = typename E::storage;
  constexpr bool HALF = sizeof(S) == 2;
  constexpr int WORDS = HALF ? 8 : 16;
  struct alignas(16) Vec { uint32_t w[WORDS]; };
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  const uint32_t block = item / (uint32_t)a.groups;
  const int g = (int)(item - block * (uint32_t)a.groups);
  const int64_t t0 = (int64_t)block * ROWS;
  if (t0 >= a.T) return;  // whole 8-lane groups leave together
  const int k = g * 128 + l * 16;
  // (unconditional, past the end the last again: a load in a branch of its own would be waited for there)
  const S* x = static_cast<const S*>(a.x) + (k < a.K ? k : 0);
  Vec in[ROWS];
#pragma unroll
  for (int j = 0; j < ROWS; ++j) in[j] = *reinterpret_cast<const Vec*>(x + min(t0 + j, (int64_t)a.T - 1) * a.x_stride);
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {
    if (j > 0 && t0 + j >= a.T) break;
    float v[16];
    uint32_t m = 0;
    float v_least;  // the smallest magnitude but 0
    if (k >= a.K) in[j] = Vec{};
    if constexpr (HALF) {  // magnitudes of 16-bit values order as their bits do, two at a time
      u16x2 most = {0, 0}, least = {0xFFFF, 0xFFFF};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t w = in[j].w[i];
        const u16x2 mag = __builtin_bit_cast(u16x2, w & 0x7FFF7FFFu);
        most = __builtin_elementwise_max(most, mag);
        least = __builtin_elementwise_min(least, (u16x2)(mag - (u16x2){1, 1}));
        v[2 * i] = E::to_float((uint16_t)w);
        v[2 * i + 1] = E::to_float((uint16_t)(w >> 16));
      }
      m = __builtin_bit_cast(uint32_t, E::to_float(max(most[0], most[1])));
      const uint16_t one = min(least[0], least[1]);  // the smallest but 0, less one; 0xFFFF: none
      v_least = one == 0xFFFF ? INFINITY : E::to_float((uint16_t)(one + 1));
    } else {
      uint32_t least = ~0u;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        v[i] = __builtin_bit_cast(float, in[j].w[i]);
        m = max(m, in[j].w[i] & 0x7FFFFFFFu);
        least = min(least, (in[j].w[i] & 0x7FFFFFFFu) - 1u);
      }
      v_least = least == ~0u ? INFINITY : __builtin_bit_cast(float, least + 1u);
    }
    // over the 8 lanes, by DPP moves: the xor of 1 and 2, a mirror of 8
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xf, 0xf, true));
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xf, 0xf, true));
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xf, 0xf, true));
    const float s = quant_scale(m), r = 1.0f / s;
    const int64_t t = t0 + j;
    if (k < a.K) {
      float q[16];
      quant_values(v, s, r, v_least < s * QUANT_LOW, q);
      *reinterpret_cast<u32x4_t*>(a.out + t * a.out_stride + k) =
          u32x4_t{fp8_pack4(q), fp8_pack4(q + 4), fp8_pack4(q + 8), fp8_pack4(q + 12)};
    }
    if (l == 0) a.scale[t * a.scale_row + g * a.scale_grp] = s;
  }
}
// rows below each other once that still leaves eight workgroups of 32 groups to a CU
inline int quant_rows(int64_t T, int groups) { return T * groups >= 2ll * 32 * 8 * 256 ? 2 : 1; }

template <int DT> __device__ inline mm4_t mm_mma(u32x4_t a, u32x4_t b, mm4_t c) {
  if constexpr (DT == GR_DTYPE_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                   0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0,
                                                  0, 0);
}

// four neighbouring results in the output's type
template <int OT> __device__ __forceinline__ void mm_store(void* out, int64_t at, const float (&v)[4]) {
  if constexpr (OT == GR_DTYPE_F32)
    *reinterpret_cast<mm4_t*>(static_cast<float*>(out) + at) = mm4_t{v[0], v[1], v[2], v[3]};
  else
    *reinterpret_cast<u32x2_t*>(static_cast<uint16_t*>(out) + at) =
        u32x2_t{Mma<OT>::pack2(v[0], v[1]), Mma<OT>::pack2(v[2], v[3])};
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

// One 16-byte chunk per lane of a buffer (base and length in d) into LDS: lane i's,
// from byte off + soff, lands at lds + 16 i; zeros where off is past the length.  (M0
// is no value's home for the compiler: it sets it where an instruction of its own reads it.)
__device__ __forceinline__ void dma_b(uint32_t lds, u32x4_t d, uint32_t off, uint32_t soff) {
  __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                   : : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(off), "s"(d), "s"(__builtin_amdgcn_readfirstlane(soff))
               : "memory");
}
// A buffer of 2 GB from p on: offsets of MM_NOWHERE and more read zeros.
constexpr uint32_t MM_NOWHERE = 0x80000000u;
__device__ inline u32x4_t mm_buffer(const void* p) {
  const uint64_t b = reinterpret_cast<uint64_t>(p);
  return u32x4_t{(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)b),
                 (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(b >> 32)) & 0xFFFFu, MM_NOWHERE, 0x00027000u};
}

// What a tile's workgroup knows about it.
struct MmTile {
  int mt, nt, m0, m_end, n0;
  const uint8_t* w;
  const float* ws;
};

// XT: element type of both operands.  WM x WN waves over a BM x BN tile (BN weight
// rows; with SwiGLU 16 gate rows and the 16 up rows of the same columns alternate).
template <int XT, int BM, int BN, int WM, int WN, int MODE, bool EXPERTS, bool EXACT>
struct Mm {
  static constexpr bool F8 = XT == GR_DTYPE_FP8_E4M3;
  static constexpr bool GATED = MODE == MM_SWIGLU || MODE == MM_SWIGLU_Q;
  static constexpr bool QUANT = MODE == MM_SWIGLU_Q || MODE == MM_PLAIN_Q;
  static constexpr int NW = WM * WN;
  static constexpr int TILE = (BM + BN) * 128;              // bytes of a stage
  static constexpr int SCALES = F8 ? NW * 256 : 0;          // and of its scales
  static constexpr int LPS = (BM + BN) / 8 / NW;            // transfers per wave and stage, 8 rows each
  static constexpr int OPS = LPS + (F8 ? 1 : 0);
  static constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
  static constexpr int OC = GATED ? BN / 2 : BN;            // output columns of the tile
  static constexpr int WBLOCKS = (OC + 127) / 128 * (GATED ? 2 : 1);  // weight blocks of the tile
  static_assert(F8 || !EXACT, "16-bit sums are exact as they are");
  static_assert(BM % (16 * WM) == 0 && BN % (16 * WN) == 0 && (!GATED || FN % 2 == 0), "whole fragments");
  static_assert(OC / WN <= 128 && 128 % (OC / WN) == 0 && (OC / WN) % 16 == 0, "a wave's columns share a weight block");
  static_assert(!QUANT || OC == 128, "a tile's columns are one group of the result");

  using Acc = mm4_t[FN][FM];

  // Transfer i of a stage moves LDS rows 8 (wave + NW i) .. + 7 (x rows, then w
  // rows); lane l lands on row l >> 3, chunk l & 7 of them and fetches the logical
  // chunk (l & 7) ^ (row & 7).  Rows past the tile's last repeat it (their results
  // are not stored).  One more transfer, of a dword a lane, moves the scales.
  struct Source {
    u32x4_t buf[LPS];   // wave-uniform
    uint32_t off[LPS];
    const float* scale;
    int scale_step;
    uint32_t ch;        // this lane's byte within a stage of a row
  };

  __device__ static __forceinline__ bool tile(const MmArgs& a, MmTile& t) {
    const int tiles_m = EXPERTS ? __builtin_amdgcn_readfirstlane(*a.num_tiles) : a.tiles_m;
    if (!mm_tile(a, tiles_m, t.mt, t.nt)) return false;
    t.m0 = t.mt * BM;
    t.m_end = a.M;
    t.w = a.w;
    t.ws = a.ws;
    if constexpr (EXPERTS) {
      const int4 e = a.tiles[t.mt];
      const int id = __builtin_amdgcn_readfirstlane(e.x);
      t.m0 = __builtin_amdgcn_readfirstlane(e.y);
      t.m_end = t.m0 + __builtin_amdgcn_readfirstlane(e.z);
      t.w += id * a.w_expert;
      if constexpr (F8) t.ws += id * a.ws_expert;
    }
    t.n0 = t.nt * OC;
    return true;
  }

  __device__ static __forceinline__ int x_row(const MmArgs& a, const MmTile& t, int r) {
    const int p = min(t.m0 + r, t.m_end - 1);
    if constexpr (EXPERTS) return a.gather ? a.slot[p] / a.gather : p;
    else return p;
  }

  __device__ static __forceinline__ void source(const MmArgs& a, const MmTile& t, int wave, int lane, Source& s) {
    s.ch = ((lane & 7) ^ (lane >> 3)) * 16;
    // x rows are addressed from the tile's first one, gathered ones from the tensor's
    const int first = EXPERTS && a.gather ? 0 : t.m0;
    const u32x4_t xb = mm_buffer(a.x + (int64_t)first * a.x_stride);
    const u32x4_t wb = mm_buffer(t.w + (int64_t)t.n0 * a.w_stride);
    const u32x4_t ub = GATED ? mm_buffer(t.w + (int64_t)(t.n0 + a.N) * a.w_stride) : wb;
#pragma unroll
    for (int i = 0; i < LPS; ++i) {
      const int r8 = 8 * (wave + NW * i), row = r8 + (lane >> 3);
      if (r8 < BM) {
        s.buf[i] = xb;
        s.off[i] = (uint32_t)((x_row(a, t, row) - first) * (uint32_t)a.x_stride) + s.ch;
      } else {
        const int b = row - BM, n = GATED ? (b >> 5) * 16 + (b & 15) : b;
        s.buf[i] = GATED && ((r8 - BM) >> 4 & 1) ? ub : wb;
        s.off[i] = (uint32_t)(min(n, a.N - 1 - t.n0) * (uint32_t)a.w_stride) + s.ch;
      }
    }
    if constexpr (F8) {
      // entries: the tile's rows, then its weight blocks (with SwiGLU gate's, then up's)
      const int e = wave * 64 + lane, kb = (a.kbytes + 127) >> 7, nb = (a.N + 127) >> 7;
      if (e < BM || e >= BM + WBLOCKS) {
        s.scale = a.xs + x_row(a, t, min(e, BM - 1)) * a.xs_row;
        s.scale_step = (int)a.xs_grp;
      } else {
        constexpr int HALF = WBLOCKS / (GATED ? 2 : 1);
        const int up = GATED ? (e - BM) / HALF : 0;
        s.scale = t.ws + (int64_t)(up * nb + min((t.n0 >> 7) + (e - BM) % HALF, nb - 1)) * kb;
        s.scale_step = 1;
      }
    }
  }

  // Stage k of a tile into the buffer at LDS byte `lds`, its scales to `sc`.
  __device__ static __forceinline__ void fetch(const MmArgs& a, const Source& s, int k, uint32_t lds, uint32_t sc, int wave) {
    if ((k + 1) * 128 <= a.kbytes) {
#pragma unroll
      for (int i = 0; i < LPS; ++i) dma_b(lds + (uint32_t)(wave + NW * i) * 1024, s.buf[i], s.off[i], (uint32_t)k * 128);
    } else {  // a short last stage: zeros behind its end
      const bool in = k * 128 + (int)s.ch < a.kbytes;
#pragma unroll
      for (int i = 0; i < LPS; ++i)
        dma_b(lds + (uint32_t)(wave + NW * i) * 1024, s.buf[i], in ? s.off[i] : MM_NOWHERE, (uint32_t)k * 128);
    }
    if constexpr (F8) dma_v1(sc + wave * 256, s.scale + (int64_t)k * s.scale_step);
  }

  struct Lane {
    int xo, wo, fch[2], so, wso[GATED ? 2 : 1];
  };
  __device__ static __forceinline__ Lane lane_of(int wm, int wn, int lane) {
    const int r16 = lane & 15, q = lane >> 4;
    Lane l;
    l.fch[0] = (q ^ (r16 & 7)) * 16;
    l.fch[1] = ((4 + q) ^ (r16 & 7)) * 16;
    l.xo = (wm * (BM / WM) + r16) * 128;
    l.wo = (BM + wn * (BN / WN) + r16) * 128;
    l.so = (wm * (BM / WM) + r16) * 4;
    l.wso[0] = (BM + (wn * (OC / WN)) / 128) * 4;
    if constexpr (GATED) l.wso[1] = l.wso[0] + WBLOCKS / 2 * 4;
    return l;
  }
  // a lane's 32 bytes of a fragment of 16 rows: one 8-bit operand, or two 16-bit ones
  __device__ static __forceinline__ mm8i_t read(const uint8_t* p, const Lane& l) {
    const mm4i_t a = *reinterpret_cast<const mm4i_t*>(p + l.fch[0]), b = *reinterpret_cast<const mm4i_t*>(p + l.fch[1]);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  // the wave's weight fragments and their blocks' scales
  __device__ static __forceinline__ void read_w(const uint8_t* p, const uint8_t* sc, const Lane& l, mm8i_t (&w)[FN],
                                                float (&ws)[2]) {
#pragma unroll
    for (int i = 0; i < FN; ++i) w[i] = read(p + l.wo + i * 2048, l);
    ws[0] = ws[1] = 0.f;
    if constexpr (F8) {
      ws[0] = *reinterpret_cast<const float*>(sc + l.wso[0]);
      if constexpr (GATED) ws[1] = *reinterpret_cast<const float*>(sc + l.wso[1]);
    }
  }
  __device__ static __forceinline__ u32x4_t half(mm8i_t v, int h) {
    return __builtin_bit_cast(u32x4_t, h ? __builtin_shufflevector(v, v, 4, 5, 6, 7)
                                         : __builtin_shufflevector(v, v, 0, 1, 2, 3));
  }
  // fragment bytes 8 z .. + 7 as fp16
  __device__ static __forceinline__ u32x4_t fp16(mm8i_t v, int z) {
    return Fp8Cvt<GR_DTYPE_F16>::x8((uint32_t)v[2 * z], (uint32_t)v[2 * z + 1]);
  }
  __device__ static __forceinline__ void convert(const mm8i_t (&w)[FN], u32x4_t (&wh)[4][FN]) {
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int z = 0; z < 4; ++z) wh[z][i] = fp16(w[i], z);
  }
  // products of fragment row j; xs, ws0, ws1: the row's scale and the weight blocks'
  __device__ static __forceinline__ void mul(const mm8i_t (&w)[FN], mm8i_t x, int j, float xs, float ws0, float ws1,
                                             Acc& acc) {
    if constexpr (F8 && !EXACT) {
      const float c0 = xs * ws0, c1 = GATED ? xs * ws1 : c0;
#pragma unroll
      for (int i = 0; i < FN; ++i) {
        const mm4_t z = {0.f, 0.f, 0.f, 0.f};
        const mm4_t t = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w[i], x, z, 0, 0, 0, 0, 0, 0);
        const float c = GATED && (i & 1) ? c1 : c0;
#pragma unroll
        for (int u = 0; u < 4; ++u) acc[i][j][u] = fmaf(t[u], c, acc[i][j][u]);
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < FN; ++i) acc[i][j] = mm_mma<XT>(half(w[i], h), half(x, h), acc[i][j]);
    }
  }
  // the same with the operands converted to fp16; wh: fragment bytes 8 z .. + 7 of the weights
  __device__ static __forceinline__ void mul_exact(const u32x4_t (&wh)[4][FN], mm8i_t x, int j, float xs, float ws0,
                                                   float ws1, Acc& acc) {
    const float c0 = xs * ws0, c1 = GATED ? xs * ws1 : c0;
    u32x4_t xh[4];
#pragma unroll
    for (int z = 0; z < 4; ++z) xh[z] = fp16(x, z);
    mm4_t t[FN];
#pragma unroll
    for (int i = 0; i < FN; ++i) t[i] = mm4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int z = 0; z < 4; ++z)
#pragma unroll
      for (int i = 0; i < FN; ++i) t[i] = mm_mma<GR_DTYPE_F16>(wh[z][i], xh[z], t[i]);
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int u = 0; u < 4; ++u) acc[i][j][u] = fmaf(t[i][u], GATED && (i & 1) ? c1 : c0, acc[i][j][u]);
  }

  // a stage's operands in registers
  struct Frags {
    mm8i_t w[FN], x[FM];
    float ws[2], xs[FM];
  };
  __device__ static __forceinline__ void read_all(const uint8_t* p, const uint8_t* sc, const Lane& l, Frags& f) {
    read_w(p, sc, l, f.w, f.ws);
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      f.x[j] = read(p + l.xo + j * 2048, l);
      f.xs[j] = F8 ? *reinterpret_cast<const float*>(sc + l.so + j * 64) : 0.f;
    }
  }
  __device__ static __forceinline__ void mul_all(const Frags& f, Acc& acc) {
#pragma unroll
    for (int j = 0; j < FM; ++j) mul(f.w, f.x[j], j, f.xs[j], f.ws[0], f.ws[1], acc);
  }

  // fragment (i, j), register u: column 16 i + 4 (lane / 16) + u, row 16 j + lane % 16
  // (the gate by the reciprocal instruction, an ulp off, where a division is ten instructions: with the results taken
  // once, not for the largest and again for the rounding, 512 x 6144 quantised of 2048 features 37.8 us from 41.2)
  static constexpr int FO = FN / (GATED ? 2 : 1);  // output fragments
  __device__ static __forceinline__ void value(const Acc& acc, int i, int j, float (&v)[4]) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if constexpr (GATED) {
        const float g = acc[2 * i][j][u];
        // (g sigmoid(g) = 2^-7 g / (2^-7 + 2^(-g log2(e) - 7)): neither the power nor its reciprocal leaves the normal
        // numbers before the product does, at a gate of -91.8)
        const float e = __builtin_amdgcn_exp2f(fmaf(g, -LOG2E, -7.0f));
        v[u] = g * 0x1p-7f * __builtin_amdgcn_rcpf(e + 0x1p-7f) * acc[2 * i + 1][j][u];
      } else {
        v[u] = acc[i][j][u];
      }
    }
  }
  __device__ static __forceinline__ int64_t out_row(const MmArgs& a, const MmTile& t, int r) {
    if constexpr (EXPERTS) return a.scatter ? a.slot[t.m0 + r] : t.m0 + r;
    else return t.m0 + r;
  }

  // Results of one wave: through LDS (its own part, a fragment row at a time), so that
  // whole lines are written instead of 16 pieces of 32 bytes each -- 8192 x 8192 bf16
  // results of 2048 features, 142 us against 157; float32, 248 against 281.
  // The rows they go to are looked up together, and a tile that is whole (FULL) asks for
  // no row's or column's end: 65536 x 2048 results of experts of 768 270 us from 292.
  template <int OT>
  __device__ static __forceinline__ void store(const MmArgs& a, const MmTile& t, const Acc& acc, int wave, int wm, int wn,
                                               int lane, uint8_t* lds) {
    constexpr int PER = OT == GR_DTYPE_F32 ? 4 : 8;
    const bool wide = a.out_stride % PER == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;
    if (wide && t.m0 + BM <= t.m_end && t.n0 + OC <= a.N) store_rows<OT, true>(a, t, acc, wave, wm, wn, lane, lds, true);
    else store_rows<OT, false>(a, t, acc, wave, wm, wn, lane, lds, wide);
  }
  template <int OT, bool FULL>
  __device__ static __forceinline__ void store_rows(const MmArgs& a, const MmTile& t, const Acc& acc, int wave, int wm,
                                                    int wn, int lane, uint8_t* lds, bool wide) {
    constexpr bool SCALED = OT == MM_OUT_SCALED;
    using S = typename Elem<SCALED ? GR_DTYPE_F16 : OT>::storage;
    constexpr int COLS = OC / WN, PITCH = COLS * sizeof(S) + 16;  // (16: rows start on different banks)
    constexpr int PER = 16 / sizeof(S), LANES = COLS / PER;      // results a lane stores, lanes a row
    constexpr int EACH = (16 * LANES + 63) / 64;
    const int r16 = lane & 15, q = lane >> 4, c0 = t.n0 + wn * COLS, last = t.m_end - t.m0 - 1;
    uint8_t* mine = lds + wave * 16 * PITCH;
    int64_t to[FM][EACH], to16[FM];
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      const int r0 = wm * (BM / WM) + j * 16;
#pragma unroll
      for (int e = 0; e < EACH; ++e) to[j][e] = out_row(a, t, min(r0 + (64 * e + lane) / LANES, last));
      if constexpr (SCALED) to16[j] = out_row(a, t, min(r0 + r16, last));
    }
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      const int r0 = wm * (BM / WM) + j * 16;
      if (!FULL && r0 > last) break;
      float unit = 1.f;
      if constexpr (SCALED) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < FO; ++i) {
          float v[4];
          value(acc, i, j, v);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const uint32_t b = __builtin_bit_cast(uint32_t, v[u]) & 0x7FFFFFFFu;
            m = max(m, b < 0x7F800000u ? b : 0u);
          }
        }
        m = max(m, (uint32_t)__shfl_xor((int)m, 16, 64));
        m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
        // (a largest below 2^-98 keeps the unit of that)
        const int e = max((int)(m >> 23) - 127, -98) - 14;
        unit = __builtin_bit_cast(float, (uint32_t)(127 - e) << 23);
        if (q == 0 && (FULL || (r0 + r16 <= last && c0 < a.N)))
          a.out_exp[to16[j] * ((a.N + COLS - 1) / COLS) + c0 / COLS] = (int8_t)e;
      }
#pragma unroll
      for (int i = 0; i < FO; ++i) {
        float v[4];
        value(acc, i, j, v);
        if constexpr (SCALED)
#pragma unroll
          for (int u = 0; u < 4; ++u) v[u] *= unit;
        S* o = reinterpret_cast<S*>(mine + r16 * PITCH) + 16 * i + 4 * q;
        if constexpr (OT == GR_DTYPE_F32) *reinterpret_cast<mm4_t*>(o) = mm4_t{v[0], v[1], v[2], v[3]};
        else *reinterpret_cast<u32x2_t*>(o) = u32x2_t{Mma<SCALED ? GR_DTYPE_F16 : OT>::pack2(v[0], v[1]),
                                                      Mma<SCALED ? GR_DTYPE_F16 : OT>::pack2(v[2], v[3])};
      }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        const int r = (64 * e + lane) / LANES, col = (64 * e + lane) % LANES * PER;
        if (16 * LANES < 64 && lane >= 16 * LANES) continue;
        const u32x4_t d = *reinterpret_cast<const u32x4_t*>(mine + r * PITCH + col * sizeof(S));
        if (!FULL && (r0 + r > last || c0 + col >= a.N)) continue;
        S* o = static_cast<S*>(a.out) + to[j][e] * a.out_stride + c0 + col;
        if (FULL || (wide && c0 + col + PER <= a.N)) {
          *reinterpret_cast<u32x4_t*>(o) = d;
        } else {
          struct { S e[PER]; } p = __builtin_bit_cast(decltype(p), d);
#pragma unroll
          for (int u = 0; u < PER; ++u)
            if (c0 + col + u < a.N) o[u] = p.e[u];
        }
      }
      __builtin_amdgcn_wave_barrier();
    }
  }

  // The results; `lds` may be overwritten once every wave is here.
  __device__ static __forceinline__ void finish(const MmArgs& a, const MmTile& t, const Acc& acc, int wave, int wm, int wn,
                                                int lane, uint8_t* lds) {
    __syncthreads();
    if constexpr (QUANT) {
      // the group's largest value: over the lane's columns, the four lanes of the
      // row, then the waves of the row through LDS
      constexpr int PITCH = 128 + 16;
      const int r16 = lane & 15, q = lane >> 4, c0 = wn * (OC / WN) + 4 * q;
      uint32_t* part = reinterpret_cast<uint32_t*>(lds);  // [WN][BM]
      uint8_t* rows = lds + WN * BM * 4;                  // [BM][PITCH]
      float v[FM][FO * 4];
#pragma unroll
      for (int j = 0; j < FM; ++j) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < FO; ++i) {
          float y[4];
          value(acc, i, j, y);
          const bool in = t.n0 + c0 + 16 * i < a.N;
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            v[j][4 * i + u] = in ? y[u] : 0.f;
            m = max(m, __builtin_bit_cast(uint32_t, v[j][4 * i + u]) & 0x7FFFFFFFu);
          }
        }
        m = max(m, (uint32_t)__shfl_xor((int)m, 16, 64));
        m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
        if (q == 0) part[wn * BM + wm * (BM / WM) + j * 16 + r16] = m;
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < FM; ++j) {
        const int r = wm * (BM / WM) + j * 16 + r16;
        uint32_t m = 0;
#pragma unroll
        for (int k = 0; k < WN; ++k) m = max(m, part[k * BM + r]);
        const float s = quant_scale(m), rs = 1.0f / s;
        if (wn == 0 && q == 0 && t.m0 + r < t.m_end) a.out_scale[out_row(a, t, r) * a.os_row + t.nt * a.os_grp] = s;
        float z[FO * 4];
        quant_values(v[j], s, rs, quant_low(v[j], s), z);
#pragma unroll
        for (int i = 0; i < FO; ++i) *reinterpret_cast<uint32_t*>(rows + r * PITCH + c0 + 16 * i) = fp8_pack4(z + 4 * i);
      }
      __syncthreads();
      // whole rows of 128 bytes
      const bool wide = a.out_stride % 16 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;
      const int ch = (lane & 7) * 16;
      for (int r = wave * 8 + (lane >> 3); r < BM; r += NW * 8) {
        if (t.m0 + r >= t.m_end || t.n0 + ch >= a.N) continue;  // (N is a multiple of 16)
        const u32x4_t d = *reinterpret_cast<const u32x4_t*>(rows + r * PITCH + ch);
        uint8_t* o = static_cast<uint8_t*>(a.out) + out_row(a, t, r) * a.out_stride + t.n0 + ch;
        if (wide) {
          *reinterpret_cast<u32x4_t*>(o) = d;
        } else {
#pragma unroll
          for (int u = 0; u < 4; ++u) reinterpret_cast<uint32_t*>(o)[u] = d[u];
        }
      }
    } else {
      store_any(a, t, acc, wave, wm, wn, lane, lds);
    }
  }
  __device__ static __forceinline__ void store_any(const MmArgs& a, const MmTile& t, const Acc& acc, int wave, int wm, int wn,
                                                   int lane, uint8_t* lds) {
    if constexpr (EXPERTS && MODE == MM_PLAIN) {
      if (a.out_type == MM_OUT_SCALED) return store<MM_OUT_SCALED>(a, t, acc, wave, wm, wn, lane, lds);
      return store<GR_DTYPE_F32>(a, t, acc, wave, wm, wn, lane, lds);
    }
    if (a.out_type == GR_DTYPE_BF16) store<GR_DTYPE_BF16>(a, t, acc, wave, wm, wn, lane, lds);
    else if (a.out_type == GR_DTYPE_F16) store<GR_DTYPE_F16>(a, t, acc, wave, wm, wn, lane, lds);
    else store<GR_DTYPE_F32>(a, t, acc, wave, wm, wn, lane, lds);
  }
};

// One barrier a stage: each wave reads a stage's fragments and multiplies, ST - 1
// stages on their way.  AHEAD (64 x 64 tiles): a stage's fragments are read while the
// one before multiplies, from registers, and all ST buffers are on their way: 5 to 9 %
// there (64 x 4096 by 2048 features 8.5 us against 9.0), nothing or less on larger
// tiles, whose two sets of fragments crowd the registers.
template <int XT, int BM, int BN, int WM, int WN, int ST, int MODE, bool EXPERTS, bool EXACT, bool AHEAD>
__global__ __launch_bounds__(64 * WM * WN, 2) void block_mm(MmArgs a) {
  using M = Mm<XT, BM, BN, WM, WN, MODE, EXPERTS, EXACT>;
  static_assert((BM + BN) % (8 * M::NW) == 0 && BM + M::WBLOCKS <= M::NW * 64, "whole transfers");
  static_assert(!M::QUANT || WN * BM * 4 + BM * 144 <= ST * M::TILE, "the epilogue's rows fit");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[ST * (M::TILE + M::SCALES)];
  MmTile t;
  if (!M::tile(a, t)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  typename M::Source src;
  M::source(a, t, wave, lane, src);
  const typename M::Lane l = M::lane_of(wm, wn, lane);
  const uint32_t lds0 = (uint32_t)reinterpret_cast<uintptr_t>(lds);
  const int n = __builtin_amdgcn_readfirstlane((a.kbytes + 127) >> 7);
  auto fetch = [&](int s, int buf) __attribute__((always_inline)) {
    M::fetch(a, src, s, lds0 + buf * M::TILE, lds0 + ST * M::TILE + buf * M::SCALES, wave);
  };
  typename M::Acc acc;
#pragma unroll
  for (int i = 0; i < M::FN; ++i)
#pragma unroll
    for (int j = 0; j < M::FM; ++j) acc[i][j] = mm4_t{0.f, 0.f, 0.f, 0.f};
  if constexpr (AHEAD) {
#pragma unroll
    for (int s = 0; s < ST; ++s)
      if (s < n) fetch(s, s);
    if (ST <= n) mm_wait_barrier<(ST - 1) * M::OPS>();
    else mm_wait_barrier<0>();
    typename M::Frags f0, f1;
    M::read_all(lds, lds + ST * M::TILE, l, f0);
    int buf = 0;
    // stage s is in registers; past the barrier its buffer is free, stage s + 1 has
    // landed, and stages s + 2 .. s + ST - 1 may be on their way
    auto step = [&](int s, const typename M::Frags& cur, typename M::Frags& nxt) __attribute__((always_inline)) {
      const int next = buf + 1 == ST ? 0 : buf + 1;
      if (s + 1 < n) {
        if (s + ST <= n) mm_wait_barrier<(ST - 2) * M::OPS>();
        else mm_wait_barrier<0>();
        M::read_all(lds + next * M::TILE, lds + ST * M::TILE + next * M::SCALES, l, nxt);
        if (s + ST < n) fetch(s + ST, buf);
      }
      buf = next;
      M::mul_all(cur, acc);
    };
    for (int s = 0; s < n; s += 2) {
      step(s, f0, f1);
      if (s + 1 < n) step(s + 1, f1, f0);
    }
  } else {
    // stage s has landed when all but the ST - 2 younger ones' transfers have; past
    // its barrier nobody reads stage s - 1, whose buffer takes stage s + ST - 1
#pragma unroll
    for (int s = 0; s < ST - 1; ++s)
      if (s < n) fetch(s, s);
    int buf = 0;
    for (int s = 0; s < n; ++s) {
      if (s + ST - 1 <= n) mm_wait_barrier<(ST - 2) * M::OPS>();
      else mm_wait_barrier<0>();
      if (s + ST - 1 < n) fetch(s + ST - 1, buf == 0 ? ST - 1 : buf - 1);
      const uint8_t *p = lds + buf * M::TILE, *sc = lds + ST * M::TILE + buf * M::SCALES;
      mm8i_t w[M::FN];
      u32x4_t wh[4][EXACT ? M::FN : 1];
      float ws[2];
      M::read_w(p, sc, l, w, ws);
      if constexpr (EXACT) M::convert(w, wh);
#pragma unroll
      for (int j = 0; j < M::FM; ++j) {
        const float xs = M::F8 ? *reinterpret_cast<const float*>(sc + l.so + j * 64) : 0.f;
        const mm8i_t x = M::read(p + l.xo + j * 2048, l);
        if constexpr (EXACT) M::mul_exact(wh, x, j, xs, ws[0], ws[1], acc);
        else M::mul(w, x, j, xs, ws[0], ws[1], acc);
      }
      buf = buf + 1 == ST ? 0 : buf + 1;
    }
  }
  M::finish(a, t, acc, wave, wm, wn, lane, lds);
}

// Few rows: BM = 16 FM.  What bounds this is the weights' way from memory (or, for a
// single projection, one round trip), so nothing is shared through LDS: every weight
// is loaded once, by the one wave that multiplies it, straight into the registers of
// the operand, U stages at a time, and the eight waves of 16 columns split the depth
// (wave k takes stages k, k + 8, ...).  Their partial sums meet in LDS.  The rows are
// read by every workgroup, from L2.
template <int XT, int FM, int MODE, bool EXPERTS>
__global__ __launch_bounds__(512) void few_mm(MmArgs a) {
  constexpr bool F8 = XT == GR_DTYPE_FP8_E4M3;
  constexpr bool GATED = MODE == MM_SWIGLU;
  constexpr int WK = 8, FN = GATED ? 2 : 1, U = FM == 1 ? 4 : 2;
  using M = Mm<XT, 16 * FM, 16 * FN, 1, 1, MODE, EXPERTS, F8>;
  using M1 = Mm<XT, 16, 16 * FN, 1, 1, MODE, EXPERTS, F8>;  // one fragment row
  static_assert(MODE == MM_PLAIN || MODE == MM_SWIGLU, "results that are not quantised");
  constexpr int LDS = WK * FM * FN * 1024 + 8 * 16 * 80;
  __shared__ __attribute__((aligned(16))) uint8_t lds[LDS];
  MmTile t;
  if (!M::tile(a, t)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, q = lane >> 4;
  const int n = (a.kbytes + 127) >> 7, nb = (a.N + 127) >> 7;
  const int col = min(t.n0 + r16, a.N - 1);
  const uint8_t* w0 = t.w + (int64_t)col * a.w_stride + q * 16;
  const int64_t up = (int64_t)a.N * a.w_stride;
  const float* ws = F8 ? t.ws + (int64_t)min(t.n0 >> 7, nb - 1) * n : nullptr;
  const uint8_t* x0[FM];
  const float* xs[FM];
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    const int64_t r = M::x_row(a, t, 16 * j + r16);
    x0[j] = a.x + r * a.x_stride + q * 16;
    xs[j] = F8 ? a.xs + r * a.xs_row : nullptr;
  }
  auto load = [&](const uint8_t* p, int s) __attribute__((always_inline)) {
    mm4i_t lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
    if (s * 128 + q * 16 < a.kbytes) lo = *reinterpret_cast<const mm4i_t*>(p + (int64_t)s * 128);
    if (s * 128 + 64 + q * 16 < a.kbytes) hi = *reinterpret_cast<const mm4i_t*>(p + (int64_t)s * 128 + 64);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  typename M::Acc acc;
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j) acc[i][j] = mm4_t{0.f, 0.f, 0.f, 0.f};
  for (int s0 = wave; s0 < n; s0 += WK * U) {
    mm8i_t w[U][FN], x[U][FM];
    float sx[U][FM], sw[U][FN];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + u * WK;  // (past the last: zeros)
#pragma unroll
      for (int i = 0; i < FN; ++i) {
        w[u][i] = load(w0 + i * up, s);
        sw[u][i] = F8 && s < n ? ws[(int64_t)i * nb * n + s] : 0.f;
      }
#pragma unroll
      for (int j = 0; j < FM; ++j) {
        x[u][j] = load(x0[j], s);
        sx[u][j] = F8 && s < n ? xs[j][(int64_t)s * a.xs_grp] : 0.f;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u && s0 + u * WK >= n) break;
      u32x4_t wh[4][F8 ? FN : 1];
      if constexpr (F8) M::convert(w[u], wh);
#pragma unroll
      for (int j = 0; j < FM; ++j)
        if constexpr (F8) M::mul_exact(wh, x[u][j], j, sx[u][j], sw[u][0], sw[u][FN - 1], acc);
        else M::mul(w[u], x[u][j], j, 0.f, 0.f, 0.f, acc);
    }
  }
  mm4_t* part = reinterpret_cast<mm4_t*>(lds);  // [wave][FM][FN][64]
#pragma unroll
  for (int j = 0; j < FM; ++j)
#pragma unroll
    for (int i = 0; i < FN; ++i) part[((wave * FM + j) * FN + i) * 64 + lane] = acc[i][j];
  __syncthreads();
  // wave j finishes fragment row j
  if (const int j = wave; j < FM) {
    typename M1::Acc sum;
#pragma unroll
    for (int i = 0; i < FN; ++i) {
      sum[i][0] = part[(j * FN + i) * 64 + lane];
#pragma unroll
      for (int k = 1; k < WK; ++k) {
        const mm4_t v = part[((k * FM + j) * FN + i) * 64 + lane];
#pragma unroll
        for (int u = 0; u < 4; ++u) sum[i][0][u] += v[u];
      }
    }
    MmTile tj = t;
    tj.m0 += 16 * j;
    if (tj.m0 < tj.m_end) M1::store_any(a, tj, sum, wave, 0, 0, lane, lds + WK * FM * FN * 1024);
  }
}

template <int XT, int BM, int BN, int WM, int WN, int ST, int MODE, bool EXPERTS, bool EXACT>
void launch_mm(MmArgs a, int tiles_m, hipStream_t stream) {
  using M = Mm<XT, BM, BN, WM, WN, MODE, EXPERTS, EXACT>;
  constexpr bool AHEAD = !EXACT && M::FM * M::FN <= 4;
  a.tiles_m = tiles_m;
  a.tiles_n = (a.N + M::OC - 1) / M::OC;
  const int64_t total = (int64_t)tiles_m * a.tiles_n;
  hipLaunchKernelGGL((block_mm<XT, BM, BN, WM, WN, ST, MODE, EXPERTS, EXACT, AHEAD>), dim3((unsigned)((total + 7) / 8 * 8)),
                     dim3(64 * WM * WN), 0, stream, a);
}

template <int XT, int FM, int MODE, bool EXPERTS>
void launch_few(MmArgs a, int tiles_m, hipStream_t stream) {
  a.tiles_m = tiles_m;
  a.tiles_n = (a.N + 15) / 16;
  const int64_t total = (int64_t)tiles_m * a.tiles_n;
  hipLaunchKernelGGL((few_mm<XT, FM, MODE, EXPERTS>), dim3((unsigned)((total + 7) / 8 * 8)), dim3(512), 0, stream, a);
}

}  // namespace
}  // namespace gr
