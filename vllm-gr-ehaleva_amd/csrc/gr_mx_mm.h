// Products of 4-bit microscaled (MXFP4) rows, and the pieces that the quantiser,
// the projections (gr_mxfp4.hip) and the experts' layers (gr_mx_experts.hip) share.
//
//   y[t, n] = sum_b 2^(xs[t, b] - 127) 2^(ws[n, b] - 127) sum_{k in block b of 32} x[t, k] w[n, k]
//
// The matrix core takes 32 numbers of e2m1 a lane and the block's two scale bytes
// beside them, and sums 128 products a result: exactly, measured, as long as the four
// blocks' scales are within 2^6 of each other, and to 2^-24 of the sum of magnitudes
// beyond.  So float32 results and results that are rounded to 4 bits again need no
// other path than 16-bit ones.
//
// A stage is 128 bytes of each row of both operands, 256 features or 8 blocks, moved
// and laid out as gr_block_mm.h does (Mm below: tiles, transfers, results); lane
// (r = l % 16, q = l / 16) of a fragment of 16 rows multiplies blocks 2 q and 2 q + 1
// of row r, so that a stage's scales are two neighbouring bytes of that row.
#pragma once

#include <type_traits>

#include "gr_block_mm.h"

namespace gr {
namespace {

// A byte's scale, as a float: 2^(byte - 127) (the conversions read 0 as 2^-127 and 255 as NaN).
__device__ inline float mx_unit(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }
// The scale byte of a block from the bits of its largest magnitude (a NaN's are the
// largest): the least 2^e with max < 7 * 2^e, that is, where the largest rounds to 6 at
// most -- from 1.75 times a power of two on the next one.
__device__ inline uint32_t mx_scale(uint32_t amax_bits) {
  if (amax_bits >= 0x7F800000u) return 255u;
  const uint32_t e = (amax_bits + 0x200000u) >> 23;
  return e < 2 ? 0u : e - 2;
}
// 8 values in 4 bits
__device__ inline uint32_t mx_codes(const float (&v)[8], float unit) {
  uint32_t c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[0], v[1], unit, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], unit, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], unit, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], unit, 3);
}

struct MxArgs : MmArgs {  // kbytes: in_features / 2; strides of x and w in bytes; out in 4 bits: out_stride in bytes
  const uint8_t* xs4;     // scale bytes of a row side by side
  int64_t xs4_row;
  const uint8_t* ws4;
  int64_t ws4_row, ws4_expert;
  uint8_t* os4;  // *_Q
  int64_t os4_row;
  int blocks;  // of a row: in_features / 32
  int scale_piece;  // bytes of a row's scales that a lane can take: 16, 4 or 1 (mx_scale_piece)
};
// What rows and their strides are whole, aligned multiples of.
inline int mx_scale_piece(const MxArgs& a) {
  const uint64_t all = (uint64_t)a.blocks | reinterpret_cast<uint64_t>(a.xs4) | (uint64_t)a.xs4_row |
                       reinterpret_cast<uint64_t>(a.ws4) | (uint64_t)a.ws4_row;
  return all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1;
}

// 16 bytes a lane from global memory into LDS: lane i's land at lds + 16 i.
__device__ __forceinline__ void dma_v4(uint32_t lds, const void* addr) {
  const uint32_t m = __builtin_amdgcn_readfirstlane(lds);
  uint32_t save;
  __asm__ volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, off\n\ts_mov_b32 m0, %0"
                   : "=&s"(save) : "s"(m), "v"(addr) : "memory");
}

// BM rows by BN weight rows, KG groups of WM x WN waves (SwiGLU: 16 gate rows and their 16 up rows alternate)
template <int BM, int BN, int WM, int WN, int KG, int CH, int MODE, bool EXPERTS>
struct Mx {
  static constexpr bool GATED = MODE == MM_SWIGLU || MODE == MM_SWIGLU_Q;
  static constexpr bool QUANT = MODE == MM_SWIGLU_Q || MODE == MM_PLAIN_Q;
  using M = Mm<GR_DTYPE_BF16, BM, BN, WM, WN, GATED ? MM_SWIGLU : MM_PLAIN, EXPERTS, false>;  // rows of bytes
  static constexpr int NW = WM * WN * KG, ROWS = BM + BN, TILE = M::TILE, LPS = ROWS / 8 / NW, FM = M::FM, FN = M::FN, OC = M::OC;
  // Scales come CH stages at a time, 16 bytes a lane or (WORDS) 4, as linear rows of 8 CH
  // bytes: a transfer costs as much as one of rows does, however little it brings (experts
  // of 5001 tokens, 256 x 256 tiles: up product 114 us by words, 99 us by 16 bytes).
  static constexpr int LANES = 2 * CH, PER = 64 / LANES, SPS = (ROWS + PER * NW - 1) / (PER * NW);
  static constexpr bool WIDE = CH >= 2;
  static constexpr int WIDE_LANES = WIDE ? CH / 2 : 1, WIDE_PER = 64 / WIDE_LANES, WIDE_ALL = (ROWS + WIDE_PER - 1) / WIDE_PER,
                       WIDE_SPS = (WIDE_ALL + NW - 1) / NW;
  static constexpr int SCALES = WIDE && WIDE_ALL * 1024 > NW * SPS * 256 ? WIDE_ALL * 1024 : NW * SPS * 256;
  static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && NW % 2 == 0, "whole transfers; a wave's rows keep their parity of 8");
  static_assert(!QUANT || OC / WN % 32 == 0, "a block of the result is one wave's");
  using Acc = typename M::Acc;

  // Chunks of 16 bytes in LDS are XORed so that the four chunks of 16 rows that a
  // fragment reads at once meet no bank twice (5.2 clocks a read of 64 lanes; with the
  // row's low bits alone, or its bits 1 to 3, 8.5).
  __device__ static __forceinline__ int swizzle(int row) { return (row & 7) ^ (row >> 3 & 1); }
  // The same for a stage's 8 bytes of scales, by 16 bytes.
  static_assert(CH == 1 || CH == 2 || CH == 4, "stages of scales");
  __device__ static __forceinline__ int scale_swizzle(int row) { return CH == 4 ? row >> 2 & 1 : 0; }

  struct Source {
    typename M::Source rows;
    const uint8_t* ws;
    int scale_row[SPS];  // of x, or (past BM) of the weights
  };
  __device__ static __forceinline__ int w_row(const MmTile& t, int b, int N) {  // weight row of tile row BM + b
    if constexpr (GATED) return min(t.n0 + (b >> 5) * 16 + (b & 15), N - 1) + (b >> 4 & 1) * N;
    else return min(t.n0 + b, N - 1);
  }
  __device__ static __forceinline__ bool wide(const MxArgs& a) { return WIDE && a.scale_piece == 16; }
  __device__ static __forceinline__ int tile_row(bool wide, int i, int wave, int lane) {  // of transfer i of scales
    return wide ? (wave + NW * i) * WIDE_PER + lane / WIDE_LANES : (wave * SPS + i) * PER + lane / LANES;
  }
  __device__ static __forceinline__ void source(const MxArgs& a, const MmTile& t, int wave, int lane, Source& s) {
    s.rows.ch = ((lane & 7) ^ swizzle(wave * 8 + (lane >> 3))) * 16;
    const int first = EXPERTS && a.gather ? 0 : t.m0;
    const u32x4_t xb = mm_buffer(a.x + (int64_t)first * a.x_stride);
    const u32x4_t wb = mm_buffer(t.w + (int64_t)t.n0 * a.w_stride);
    const u32x4_t ub = GATED ? mm_buffer(t.w + (int64_t)(t.n0 + a.N) * a.w_stride) : wb;
#pragma unroll
    for (int i = 0; i < LPS; ++i) {
      const int r8 = 8 * (wave + NW * i), row = r8 + (lane >> 3);
      if (8 * NW * i < BM) {
        // (rows behind an expert's last: zeros, that nothing is read for)
        s.rows.buf[i] = xb;
        s.rows.off[i] = EXPERTS && t.m0 + row >= t.m_end ? MM_NOWHERE
                                                         : (uint32_t)((M::x_row(a, t, row) - first) * (uint32_t)a.x_stride) + s.rows.ch;
      } else {
        const int b = row - BM;
        const bool up = GATED && ((r8 - BM) >> 4 & 1);
        s.rows.buf[i] = up ? ub : wb;
        s.rows.off[i] = (uint32_t)((w_row(t, b, a.N) - (up ? a.N : 0) - t.n0) * (uint32_t)a.w_stride) + s.rows.ch;
      }
    }
    s.ws = a.ws4;
    if constexpr (EXPERTS) s.ws += __builtin_amdgcn_readfirstlane(a.tiles[t.mt].x) * a.ws4_expert;
#pragma unroll
    for (int i = 0; i < SPS; ++i) {
      const int r = min(tile_row(wide(a), i, wave, lane), ROWS - 1);
      s.scale_row[i] = r < BM ? M::x_row(a, t, r) : w_row(t, r - BM, a.N);
    }
  }

  // Scales of stages CH c .. into the buffer at LDS byte `at` of lds.  Past a row's
  // last block its last scales stand (a NaN there is the row's anyway); the
  // numbers there are zeros.
  __device__ static __forceinline__ void fetch_scales(const MxArgs& a, const Source& s, int c, uint8_t* lds, int at, int wave,
                                                      int lane) {
    const uint32_t lds0 = (uint32_t)reinterpret_cast<uintptr_t>(lds);
    auto row = [&](int i, int r) __attribute__((always_inline)) {
      return (r < BM ? a.xs4 : s.ws) + s.scale_row[i] * (r < BM ? a.xs4_row : a.ws4_row);
    };
    if (wide(a)) {
#pragma unroll
      for (int i = 0; i < WIDE_SPS; ++i) {
        if (wave + NW * i >= WIDE_ALL) break;
        const int r = tile_row(true, i, wave, lane);
        const int b0 = 8 * CH * c + 16 * ((lane & (WIDE_LANES - 1)) ^ scale_swizzle(r));
        dma_v4(lds0 + at + (wave + NW * i) * 1024, row(i, r) + min(b0, a.blocks - 16));
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < SPS; ++i) {
      const int r = tile_row(false, i, wave, lane);
      const int b0 = 8 * CH * c + 4 * ((lane & (LANES - 1)) ^ 4 * scale_swizzle(r));
      const uint8_t* p = row(i, r);
      const int to = at + (wave * SPS + i) * 256;
      if (a.scale_piece == 1) {
        uint32_t v = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b) v |= (uint32_t)p[min(b0 + b, a.blocks - 1)] << (8 * b);
        *reinterpret_cast<uint32_t*>(lds + to + lane * 4) = v;
      } else {
        dma_v1(lds0 + to, p + min(b0, a.blocks - 4));
      }
    }
  }

  // Transfer i of stage k's rows into the buffer at LDS byte `lds`.
  __device__ static __forceinline__ void fetch_rows(const MxArgs& a, const Source& s, int i, int k, uint32_t lds, int wave) {
    const bool in = k * 128 + (int)s.rows.ch < a.kbytes;  // (a short last stage: zeros behind its end)
    dma_b(lds + (uint32_t)(wave + NW * i) * 1024, s.rows.buf[i], in ? s.rows.off[i] : MM_NOWHERE, (uint32_t)k * 128);
  }

  struct Lane {
    int xo, wo, fch[2], xso, wso, ssw;
  };
  __device__ static __forceinline__ Lane lane_of(int wm, int wn, int lane) {
    const int r16 = lane & 15, q = lane >> 4;
    Lane l;
    l.fch[0] = (2 * q ^ swizzle(r16)) * 16;
    l.fch[1] = ((2 * q + 1) ^ swizzle(r16)) * 16;
    const int xr = wm * (BM / WM) + r16, wr = BM + wn * (BN / WN) + r16;
    l.xo = xr * 128;
    l.wo = wr * 128;
    l.ssw = scale_swizzle(r16) * 16;
    l.xso = xr * (8 * CH) + 2 * q;
    l.wso = wr * (8 * CH) + 2 * q;
    return l;
  }
  struct Frag {  // a lane's two blocks of a fragment of 16 rows
    mm4i_t v[2];
    int s;
  };
  __device__ static __forceinline__ Frag read(const uint8_t* rows, const uint8_t* scale, const Lane& l) {
    return {{*reinterpret_cast<const mm4i_t*>(rows + l.fch[0]), *reinterpret_cast<const mm4i_t*>(rows + l.fch[1])},
            *reinterpret_cast<const uint16_t*>(scale)};
  }
};

// 128 features deep; H: which of a fragment's blocks
template <int H> __device__ __forceinline__ mm4_t mx_mma(mm4i_t w, int ws, mm4i_t x, int xs, mm4_t c) {
  constexpr int E2M1 = 4;
  const mm8i_t a = __builtin_shufflevector(w, w, 0, 1, 2, 3, -1, -1, -1, -1);
  const mm8i_t b = __builtin_shufflevector(x, x, 0, 1, 2, 3, -1, -1, -1, -1);
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, E2M1, E2M1, H, ws, H, xs);
}

// A 4-bit block of 32 results of row r % 16 of a fragment row: scale byte, and this
// lane's 4 + 4 codes of output fragments i and i + 1.
template <typename M> __device__ __forceinline__ uint32_t mx_block(const typename M::Acc& acc, int i, int j, uint32_t& codes) {
  float lo[4], hi[4];
  M::value(acc, i, j, lo);
  M::value(acc, i + 1, j, hi);
  const float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  uint32_t m = 0;
#pragma unroll
  for (int u = 0; u < 8; ++u) m = max(m, __builtin_bit_cast(uint32_t, v[u]) & 0x7FFFFFFFu);
  m = max(m, (uint32_t)__shfl_xor((int)m, 16, 64));
  m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
  const uint32_t s = mx_scale(m);
  codes = s == 255u ? 0u : mx_codes(v, mx_unit(s));
  return s;
}

// A step is a stage, or one for each of KG groups of waves, whose sums meet in LDS: where a
// CU has one workgroup, a group's reads and products go on while the other waits (512 x
// 2048 of 6144 features, 64 x 64 tiles 10.8 us and 9.9, 64 x 128 14.2 and 12.5).
// ST steps of LDS, one barrier a step, as block_mm: step s has landed when all but the
// ST - 2 younger ones' transfers of rows have (scales are sent ahead of their first step's
// rows, so they have too); past its barrier nobody reads step s - 1, whose buffer takes
// step s + ST - 1, nor the scales before the current ones.
template <int BM, int BN, int WM, int WN, int KG, int ST, int CH, int MODE, bool EXPERTS> struct MxLds {
  using X = Mx<BM, BN, WM, WN, KG, CH, MODE, EXPERTS>;
  static_assert(CH % KG == 0, "whole steps");
  static constexpr int STEPS = CH / KG, NS = (ST - 1 + STEPS - 1) / STEPS + 1;  // that a buffer of scales is for, and buffers
  static constexpr int BYTES = ST * KG * X::TILE + NS * X::SCALES;
  static constexpr int WAVES = X::NW / 4 * (BYTES <= 80 * 1024 ? 2 : 1);  // of a SIMD: two workgroups, where LDS has room
};
template <int BM, int BN, int WM, int WN, int KG, int ST, int CH, int MODE, bool EXPERTS>
__global__ __launch_bounds__(64 * WM * WN * KG, (MxLds<BM, BN, WM, WN, KG, ST, CH, MODE, EXPERTS>::WAVES)) void mx_mm(MxArgs a) {
  using X = Mx<BM, BN, WM, WN, KG, CH, MODE, EXPERTS>;
  using L = MxLds<BM, BN, WM, WN, KG, ST, CH, MODE, EXPERTS>;
  using M = typename X::M;
  constexpr int BLOCKS = X::OC / 32, PITCH = X::OC / 2 + 16;  // of a row in 4 bits
  constexpr int AT_SCALES = ST * KG * X::TILE;
  static_assert(!X::QUANT || BM * (PITCH + BLOCKS) <= AT_SCALES, "the results' rows fit");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[L::BYTES];
  MmTile t;
  if (!M::tile(a, t)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kg = wave / (WM * WN), wt = wave % (WM * WN), wm = wt / WN, wn = wt % WN;
  typename X::Source src;
  X::source(a, t, wave, lane, src);
  const typename X::Lane l = X::lane_of(wm, wn, lane);
  const int n = __builtin_amdgcn_readfirstlane((a.kbytes + 128 * KG - 1) / (128 * KG));
  const uint32_t lds0 = (uint32_t)reinterpret_cast<uintptr_t>(lds);
  auto scales = [&](int s) __attribute__((always_inline)) {
    if (s % L::STEPS == 0) X::fetch_scales(a, src, s / L::STEPS, lds, AT_SCALES + s / L::STEPS % L::NS * X::SCALES, wave, lane);
  };
  auto scales_at = [&](int s) __attribute__((always_inline)) {
    return lds + AT_SCALES + s / L::STEPS % L::NS * X::SCALES + ((s % L::STEPS * KG + kg) * 8 ^ l.ssw);
  };
  typename X::Acc acc;
#pragma unroll
  for (int i = 0; i < X::FN; ++i)
#pragma unroll
    for (int j = 0; j < X::FM; ++j) acc[i][j] = mm4_t{0.f, 0.f, 0.f, 0.f};
  constexpr int SENDS = KG * X::LPS;  // of a wave and step
  auto send = [&](int c, int s, uint32_t to) __attribute__((always_inline)) {
    X::fetch_rows(a, src, c % X::LPS, s * KG + c / X::LPS, to + c / X::LPS * X::TILE, wave);
  };
#pragma unroll
  for (int s = 0; s < ST - 1; ++s)
    if (s < n) {
      scales(s);
#pragma unroll
      for (int c = 0; c < SENDS; ++c) send(c, s, lds0 + s * KG * X::TILE);
    }
  int buf = 0;
  // The transfers of a step ahead are sent between the first products: sent in one go
  // they keep their wave from its products until the last is taken (512 x 2048 of 6144
  // features, 64 x 128 tiles, 17.2 us and 15.4).
  auto step = [&](int s, auto ahead) __attribute__((always_inline)) {
    constexpr bool AHEAD = decltype(ahead)::value;
    constexpr int SLOTS = X::FM * X::FN, EACH = (SENDS + SLOTS - 1) / SLOTS;
    const uint8_t *p = lds + (buf * KG + kg) * X::TILE, *sc = scales_at(s);
    const uint32_t to = lds0 + (buf == 0 ? ST - 1 : buf - 1) * KG * X::TILE;
    typename X::Frag w[X::FN], x, next;
#pragma unroll
    for (int i = 0; i < X::FN; ++i) w[i] = X::read(p + l.wo + i * 2048, sc + l.wso + i * (128 * CH), l);
    x = X::read(p + l.xo, sc + l.xso, l);
    if constexpr (AHEAD) scales(s + ST - 1);
#pragma unroll
    for (int j = 0; j < X::FM; ++j) {
      if (j + 1 < X::FM) next = X::read(p + l.xo + (j + 1) * 2048, sc + l.xso + (j + 1) * (128 * CH), l);
#pragma unroll
      for (int i = 0; i < X::FN; ++i) {
        if constexpr (AHEAD)
#pragma unroll
          for (int c = 0; c < EACH; ++c)
            if ((j * X::FN + i) * EACH + c < SENDS) send((j * X::FN + i) * EACH + c, s + ST - 1, to);
        acc[i][j] = mx_mma<0>(w[i].v[0], w[i].s, x.v[0], x.s, acc[i][j]);
        acc[i][j] = mx_mma<1>(w[i].v[1], w[i].s, x.v[1], x.s, acc[i][j]);
      }
      x = next;
    }
    buf = buf + 1 == ST ? 0 : buf + 1;
  };
  int s = 0;
  for (; s + ST - 1 < n; ++s) {
    mm_wait_barrier<(ST - 2) * SENDS>();
    step(s, std::true_type());
  }
  for (; s < n; ++s) {
    mm_wait_barrier<0>();
    step(s, std::false_type());
  }
  __syncthreads();
  if constexpr (KG > 1) {  // the groups' sums meet
    static_assert(KG == 2 && WM * WN * X::FM * X::FN * 1024 <= AT_SCALES, "room for a group's");
    mm4_t* part = reinterpret_cast<mm4_t*>(lds) + wt * X::FM * X::FN * 64 + lane;
    if (kg == 1)
#pragma unroll
      for (int i = 0; i < X::FN; ++i)
#pragma unroll
        for (int j = 0; j < X::FM; ++j) part[(i * X::FM + j) * 64] = acc[i][j];
    __syncthreads();
    if (kg == 0)
#pragma unroll
      for (int i = 0; i < X::FN; ++i)
#pragma unroll
        for (int j = 0; j < X::FM; ++j) {
          const mm4_t v = part[(i * X::FM + j) * 64];
#pragma unroll
          for (int u = 0; u < 4; ++u) acc[i][j][u] += v[u];
        }
    __syncthreads();
    if constexpr (!X::QUANT)
      if (kg == 1) return;
  }
  if constexpr (X::QUANT) {
    // through LDS, so that a row's blocks of the tile are written side by side
    const int r16 = lane & 15, q = lane >> 4, c0 = wn * (X::OC / WN);
    uint8_t* scale = lds + BM * PITCH;
#pragma unroll
    for (int j = 0; j < X::FM; ++j) {
      if (kg > 0) break;
      const int r = wm * (BM / WM) + j * 16 + r16;
#pragma unroll
      for (int g = 0; g < M::FO / 2; ++g) {
        uint32_t codes;
        const uint32_t s = mx_block<M>(acc, 2 * g, j, codes);
        uint16_t* o = reinterpret_cast<uint16_t*>(lds + r * PITCH + (c0 + 32 * g) / 2) + q;
        o[0] = (uint16_t)codes;
        o[4] = (uint16_t)(codes >> 16);
        if (q == 0) scale[r * BLOCKS + c0 / 32 + g] = (uint8_t)s;
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < BM * BLOCKS; c += 64 * X::NW) {
      const int r = c / BLOCKS, b = c % BLOCKS;
      if (t.m0 + r >= t.m_end || t.n0 + 32 * b >= a.N) continue;
      const int64_t row = M::out_row(a, t, r);
      *reinterpret_cast<u32x4_t*>(static_cast<uint8_t*>(a.out) + row * a.out_stride + t.n0 / 2 + 16 * b) =
          *reinterpret_cast<const u32x4_t*>(lds + r * PITCH + 16 * b);
      a.os4[row * a.os4_row + t.n0 / 32 + b] = scale[c];
    }
  } else if constexpr (EXPERTS) {
    M::template store<GR_DTYPE_F32>(a, t, acc, wt, wm, wn, lane, lds);
  } else {
    M::store_any(a, t, acc, wt, wm, wn, lane, lds);
  }
}

// 16 rows, 16 NF columns.  Bound by the weights' way from memory, or by one round trip:
// each weight is loaded once, by the wave that multiplies it, into the registers of the
// operand, and the WK waves split the depth (wave k takes stages k, k + WK, ...).  Their
// partial sums meet in LDS.  The rows are read by every workgroup, from L2.
template <int NF, int WK, int MODE> __global__ __launch_bounds__(64 * WK) void mx_few(MxArgs a) {
  constexpr bool GATED = MODE == MM_SWIGLU || MODE == MM_SWIGLU_Q, QUANT = MODE == MM_SWIGLU_Q || MODE == MM_PLAIN_Q;
  constexpr int FN = NF * (GATED ? 2 : 1), U = FN <= 2 ? 4 : 2;
  using M = Mm<GR_DTYPE_BF16, 16, 16 * FN, 1, 1, GATED ? MM_SWIGLU : MM_PLAIN, false, false>;
  static_assert(!QUANT || NF == 2, "a block of the result is 32 columns");
  constexpr int PART = WK * FN * 1024, ROOM = 16 * (16 * NF * 4 + 16);
  __shared__ __attribute__((aligned(16))) uint8_t lds[PART + (QUANT ? 0 : ROOM)];
  MmTile t;
  if (!M::tile(a, t)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, q = lane >> 4;
  const int n = (a.kbytes + 127) >> 7;
  const uint8_t *w0[FN], *ws[FN];
#pragma unroll
  for (int i = 0; i < FN; ++i) {
    const int64_t r = min(t.n0 + 16 * (GATED ? i >> 1 : i) + r16, a.N - 1) + (GATED && (i & 1) ? a.N : 0);
    w0[i] = t.w + r * a.w_stride + q * 32;
    ws[i] = a.ws4 + r * a.ws4_row + q * 2;
  }
  const int64_t xr = M::x_row(a, t, r16);
  const uint8_t *x0 = a.x + xr * a.x_stride + q * 32, *xs = a.xs4 + xr * a.xs4_row + q * 2;
  struct Piece {
    mm4i_t v[2];
    int s;
  };
  // (past the last block zeros, whose scale is 2^-127)
  auto load = [&](const uint8_t* p, const uint8_t* sp, int s) __attribute__((always_inline)) {
    Piece f{{{0, 0, 0, 0}, {0, 0, 0, 0}}, 0};
    const int left = a.blocks - 8 * s - 2 * q;
    if (left > 0) f.v[0] = *reinterpret_cast<const mm4i_t*>(p + (int64_t)s * 128);
    if (left > 1) {
      f.v[1] = *reinterpret_cast<const mm4i_t*>(p + (int64_t)s * 128 + 16);
      uint16_t two;
      __builtin_memcpy(&two, sp + (int64_t)s * 8, 2);
      f.s = two;
    } else if (left == 1) {
      f.s = sp[(int64_t)s * 8];
    }
    return f;
  };
  typename M::Acc acc;
#pragma unroll
  for (int i = 0; i < FN; ++i) acc[i][0] = mm4_t{0.f, 0.f, 0.f, 0.f};
  for (int s0 = wave; s0 < n; s0 += WK * U) {
    Piece w[U][FN], x[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < FN; ++i) w[u][i] = load(w0[i], ws[i], s0 + u * WK);
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = load(x0, xs, s0 + u * WK);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u && s0 + u * WK >= n) break;
#pragma unroll
      for (int i = 0; i < FN; ++i) {
        acc[i][0] = mx_mma<0>(w[u][i].v[0], w[u][i].s, x[u].v[0], x[u].s, acc[i][0]);
        acc[i][0] = mx_mma<1>(w[u][i].v[1], w[u][i].s, x[u].v[1], x[u].s, acc[i][0]);
      }
    }
  }
  mm4_t* part = reinterpret_cast<mm4_t*>(lds);  // [wave][FN][64]
#pragma unroll
  for (int i = 0; i < FN; ++i) part[(wave * FN + i) * 64 + lane] = acc[i][0];
  __syncthreads();
  if (wave == 0) {
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int k = 1; k < WK; ++k) {
        const mm4_t v = part[(k * FN + i) * 64 + lane];
#pragma unroll
        for (int u = 0; u < 4; ++u) acc[i][0][u] += v[u];
      }
    if constexpr (QUANT) {
      uint32_t codes;
      const uint32_t s = mx_block<M>(acc, 0, 0, codes);
      if (t.m0 + r16 < t.m_end) {
        const int64_t row = M::out_row(a, t, r16);
        uint16_t* o = reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(a.out) + row * a.out_stride + t.n0 / 2) + q;
        o[0] = (uint16_t)codes;
        o[4] = (uint16_t)(codes >> 16);
        if (q == 0) a.os4[row * a.os4_row + t.n0 / 32] = (uint8_t)s;
      }
    } else {
      M::store_any(a, t, acc, wave, 0, 0, lane, lds + PART);
    }
  }
}

template <int BM, int BN, int WM, int WN, int ST, int CH, int MODE, bool EXPERTS, int KG = 1>
void launch_mx(MxArgs a, int tiles_m, hipStream_t stream) {
  using X = Mx<BM, BN, WM, WN, KG, CH, MODE, EXPERTS>;
  a.tiles_m = tiles_m;
  a.tiles_n = (a.N + X::OC - 1) / X::OC;
  const int64_t total = (int64_t)tiles_m * a.tiles_n;
  hipLaunchKernelGGL((mx_mm<BM, BN, WM, WN, KG, ST, CH, MODE, EXPERTS>), dim3((unsigned)((total + 7) / 8 * 8)), dim3(64 * X::NW),
                     0, stream, a);
}
template <int NF, int WK, int MODE> void launch_mx_few(MxArgs a, hipStream_t stream) {
  a.tiles_m = (a.M + 15) / 16;
  a.tiles_n = (a.N + 16 * NF - 1) / (16 * NF);
  const int64_t total = (int64_t)a.tiles_m * a.tiles_n;
  hipLaunchKernelGGL((mx_few<NF, WK, MODE>), dim3((unsigned)((total + 7) / 8 * 8)), dim3(64 * WK), 0, stream, a);
}

// ---- rows to 4 bits ------------------------------------------------------------
struct MxQuantArgs {
  uint8_t* out;
  int64_t out_stride;  // bytes
  uint8_t* scale;
  int64_t scale_row;
  const void* x;
  int64_t x_stride;  // elements
  int T, K;
};
// N features a lane, 32 / N neighbouring lanes a block: 32 bytes of a row in one piece,
// whatever their type.  Bound by memory (8192 x 6144 bf16 22.1 us, 5.8 TB/s; two or four rows
// a lane, with their loads on their way together, 22.7 and 23.5).
template <int DT> constexpr int mx_quant_features() { return DT == GR_DTYPE_F32 ? 8 : 16; }
template <int DT> __device__ __forceinline__ void mx_quant_item(const MxQuantArgs& a, uint32_t item) {
  constexpr int N = mx_quant_features<DT>();
  struct alignas(16) Vec { uint32_t w[8]; };
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 bf2_t __attribute__((ext_vector_type(2)));
  typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
  const uint32_t per = (uint32_t)a.K / N;
  const int64_t t = item / per;
  const int k = (int)(item - (uint32_t)t * per) * N;
  if (t >= a.T) return;  // (a block's lanes leave together)
  const int64_t at = t * a.x_stride + k;
  const Vec in = DT == GR_DTYPE_F32 ? *reinterpret_cast<const Vec*>(static_cast<const float*>(a.x) + at)
                                    : *reinterpret_cast<const Vec*>(static_cast<const uint16_t*>(a.x) + at);
  uint32_t m = 0;
  if constexpr (DT == GR_DTYPE_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, in.w[i] & 0x7FFFFFFFu);
  } else {  // magnitudes of 16-bit values order as their bits do, two at a time
    u16x2 most = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, in.w[i] & 0x7FFF7FFFu));
    m = max(most[0], most[1]);
  }
  // over the block's lanes, by DPP moves: the xor of 1 (and 2)
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xf, 0xf, true));
  if constexpr (N == 8) m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xf, 0xf, true));
  if constexpr (DT != GR_DTYPE_F32) m = __builtin_bit_cast(uint32_t, Elem<DT>::to_float((uint16_t)m));
  const uint32_t s = mx_scale(m);
  const float unit = mx_unit(s);
  uint32_t c[N / 8];
  if constexpr (DT == GR_DTYPE_F32) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __builtin_bit_cast(float, in.w[i]);
    c[0] = mx_codes(v, unit);
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t* w = in.w + 4 * h;
      if constexpr (DT == GR_DTYPE_BF16) {
        c[h] = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(0u, __builtin_bit_cast(bf2_t, w[0]), unit, 0);
        c[h] = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c[h], __builtin_bit_cast(bf2_t, w[1]), unit, 1);
        c[h] = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c[h], __builtin_bit_cast(bf2_t, w[2]), unit, 2);
        c[h] = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c[h], __builtin_bit_cast(bf2_t, w[3]), unit, 3);
      } else {
        c[h] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(0u, __builtin_bit_cast(h2_t, w[0]), unit, 0);
        c[h] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c[h], __builtin_bit_cast(h2_t, w[1]), unit, 1);
        c[h] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c[h], __builtin_bit_cast(h2_t, w[2]), unit, 2);
        c[h] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c[h], __builtin_bit_cast(h2_t, w[3]), unit, 3);
      }
    }
  }
  if (s == 255u)
#pragma unroll
    for (int h = 0; h < N / 8; ++h) c[h] = 0;
  uint8_t* o = a.out + t * a.out_stride + k / 2;
  if constexpr (N == 16) *reinterpret_cast<u32x2_t*>(o) = u32x2_t{c[0], c[N / 8 - 1]};
  else *reinterpret_cast<uint32_t*>(o) = c[0];
  if (k % 32 == 0) a.scale[t * a.scale_row + k / 32] = (uint8_t)s;
}

}  // namespace
}  // namespace gr
