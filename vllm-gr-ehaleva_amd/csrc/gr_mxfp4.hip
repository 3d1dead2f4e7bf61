// 4-bit microscaled (MXFP4) tensors: rows to 4 bits and back, and the product of such
// rows with such weights (gr_mx_mm.h).
#include "gr_mx_mm.h"

#include "gr_mxfp4.h"

namespace gr {
namespace {

constexpr int MXQ_THREADS = 256;

template <int DT> __global__ __launch_bounds__(MXQ_THREADS) void mx_quant_k(MxQuantArgs a) {
  // (items: below 2^31 by the entry's check)
  mx_quant_item<DT>(a, blockIdx.x * MXQ_THREADS + threadIdx.x);
}

// ---- 4 bits to values ------------------------------------------------------------
struct MxDequantArgs {
  void* out;
  int64_t out_stride;  // elements
  const uint8_t* x;
  int64_t x_stride;  // bytes
  const uint8_t* scale;
  int64_t scale_row;
  int T, K;
};
// 8 features a lane (16 or 32 bytes of results) of two rows below each other.  Bound by
// memory, by its stores above all (8192 x 6144 bf16 23.0 us, 5.5 TB/s, and 19.9 right behind
// the quantiser, its codes in cache; one row a lane 26.7, four 24.3, eight 25.9; up to 2048 x
// 2048 none differs from another).
template <int DT> __global__ __launch_bounds__(MXQ_THREADS) void mx_dequant_k(MxDequantArgs a) {
  constexpr int ROWS = 2;
  const uint32_t item = blockIdx.x * MXQ_THREADS + threadIdx.x, per = (uint32_t)a.K / 8, band = item / per;
  const int k = (int)(item - band * per) * 8;
  const int64_t t0 = (int64_t)band * ROWS;
  if (t0 >= a.T) return;
  uint32_t c[ROWS], s[ROWS];
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {  // (past the last row: it again)
    const int64_t t = min(t0 + j, (int64_t)a.T - 1);
    c[j] = *reinterpret_cast<const uint32_t*>(a.x + t * a.x_stride + k / 2);
    s[j] = a.scale[t * a.scale_row + k / 32];
  }
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {
    if (j > 0 && t0 + j >= a.T) break;
    const float unit = mx_unit(s[j]);
    const int64_t at = (t0 + j) * a.out_stride + k;
    if constexpr (DT == GR_DTYPE_F32) {
      typedef float f32x2 __attribute__((ext_vector_type(2)));
      const f32x2 v0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[j], unit, 0), v1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[j], unit, 1),
                  v2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[j], unit, 2), v3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[j], unit, 3);
      mm4_t* o = reinterpret_cast<mm4_t*>(static_cast<float*>(a.out) + at);
      o[0] = mm4_t{v0[0], v0[1], v1[0], v1[1]};
      o[1] = mm4_t{v2[0], v2[1], v3[0], v3[1]};
    } else {
      u32x4_t v;
      if constexpr (DT == GR_DTYPE_BF16)
        v = u32x4_t{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[j], unit, 0)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[j], unit, 1)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[j], unit, 2)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c[j], unit, 3))};
      else
        v = u32x4_t{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c[j], unit, 0)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c[j], unit, 1)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c[j], unit, 2)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c[j], unit, 3))};
      *reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(a.out) + at) = v;
    }
  }
}

// ---- products ----------------------------------------------------------------------
// The tile with the least estimated time (as for the 8-bit products): over the workgroups
// of the XCD that gets the most of them, whose 32 CUs take one or two each, a round costs
// a fixed part and its stages of 256 features, `one` ns each alone on a CU, `two` with a
// neighbour.  Fitted to 339 measured sizes of 48 to 8192 rows, 512 to 12288 weight rows
// and 512 to 6144 features: the pick is 0.4 % slower than the best tile in the mean and
// 9 % at most.  (us; rows x weight rows x features, the picked tile's and the next one's)
//   400 x 4096 x 2048    64 x 64     6.9,   64 x 128   7.1
//   256 x 2048 x 6144    64 x 64, two groups  9.4, one  10.1
//   400 x 4096 x 6144    64 x 128, two groups  13.1, one  14.3
//   512 x 8192 x 2048   128 x 128   10.0,   64 x 128  10.3
//   2048 x 2048 x 6144  128 x 128   21.0,   64 x 128  25.1
//   3000 x 12288 x 512  128 x 128 of two stages, two a CU  22.0, 256 x 256  25.2
//   512 x 12288 x 2048  128 x 256   12.9,  128 x 128  13.9
//   8192 x 12288 x 2048 256 x 256    131,  128 x 128   174
struct MxChoice { int bm, bn, per_cu, launch, fixed1, one, fixed2, two; };
constexpr MxChoice kMx[] = {{64, 64, 2, 1840, 980, 296, 1500, 448},   {64, 64, 1, 1060, 1980, 249, 0, 0},  // (the second in two groups)
                            {64, 128, 2, 2060, 1310, 442, 1960, 703}, {64, 128, 1, 1240, 2560, 366, 0, 0},
                            {128, 128, 1, 910, 2690, 616, 0, 0},      {128, 128, 2, 2150, 650, 863, 2490, 1198},
                            {128, 256, 1, 550, 4290, 961, 0, 0},      {256, 256, 1, -90, 6880, 1607, 0, 0}};

int pick_mx(int M, int rows_w, int stages, bool quant) {
  int best = -1;
  int64_t least = 0;
  for (int i = quant ? 2 : 0; i < 8; ++i) {  // (a wave of a 64 x 64 tile has 16 gated results of a row, half a block)
    const MxChoice& c = kMx[i];
    const int64_t tiles = ((int64_t)((M + c.bm - 1) / c.bm) * ((rows_w + c.bn - 1) / c.bn) + 7) / 8;
    const int64_t one = c.fixed1 + (int64_t)stages * c.one, two = c.per_cu == 2 ? c.fixed2 + (int64_t)stages * c.two : one;
    const int64_t round = 32 * c.per_cu, left = tiles % round;
    const int64_t cost = c.launch + tiles / round * two + (left == 0 ? 0 : left <= 32 ? one : two);
    if (best < 0 || cost < least) {
      least = cost;
      best = i;
    }
  }
  return best;
}

// kMx' index, or below 0 the few rows' kernel of 16 (-1) or 32 (-2) columns.  Few rows, as long as the CUs hold all
// workgroups at once: 8 x 4096 x 2048 3.7 us (64 x 64 tiles 5.0), 8 x 8192 x 6144 8.5 us in 32 columns a workgroup,
// 9.5 in 16 (64 x 64 tiles 9.9; 32 x 8192 x 2048, twice that many, 7.4 and 5.2)
int pick_linear_mx(int M, int N, int kbytes, bool gated, bool quant) {
  const int64_t few = (int64_t)((M + 15) / 16) * ((N + 15) / 16);
  if (few <= 256 && !quant) return -1;
  if (few <= 512) return -2;
  return pick_mx(M, gated ? 2 * N : N, (kbytes + 127) / 128, quant);
}

template <int MODE> void launch_linear_mx(const MxArgs& a, hipStream_t stream) {
  constexpr bool GATED = MODE == MM_SWIGLU || MODE == MM_SWIGLU_Q, QUANT = MODE == MM_SWIGLU_Q || MODE == MM_PLAIN_Q;
  const int M = a.M;
  switch (pick_linear_mx(M, a.N, a.kbytes, GATED, QUANT)) {
    case -1:
      if constexpr (!QUANT) launch_mx_few<1, 8, MODE>(a, stream);
      break;
    case -2: launch_mx_few<2, 8, MODE>(a, stream); break;
    case 0:
      if constexpr (!QUANT) launch_mx<64, 64, 2, 2, 4, 4, MODE, false>(a, (M + 63) / 64, stream);
      break;
    case 1:
      if constexpr (!QUANT) launch_mx<64, 64, 2, 2, 3, 4, MODE, false, 2>(a, (M + 63) / 64, stream);
      break;
    case 2: launch_mx<64, 128, 2, 2, 3, 2, MODE, false>(a, (M + 63) / 64, stream); break;
    case 3: launch_mx<64, 128, 2, 2, 3, 4, MODE, false, 2>(a, (M + 63) / 64, stream); break;
    case 4: launch_mx<128, 128, 4, 2, 3, 2, MODE, false>(a, (M + 127) / 128, stream); break;
    case 5: launch_mx<128, 128, 4, 2, 2, 1, MODE, false>(a, (M + 127) / 128, stream); break;
    case 6: launch_mx<128, 256, 2, 4, 3, 2, MODE, false>(a, (M + 127) / 128, stream); break;
    default: launch_mx<256, 256, 2, 4, 2, 2, MODE, false>(a, (M + 255) / 256, stream);
  }
}

bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

}  // namespace
}  // namespace gr

using namespace gr;

extern "C" gr_status_t gr_quant_mxfp4(void* out, int64_t out_stride, uint8_t* scale, int64_t scale_stride, const void* x,
                                      int64_t x_stride, int num_tokens, int features, int dtype, hipStream_t stream) {
  if (num_tokens < 0 || features < 1 || !dtype_valid(dtype)) return GR_ERR_INVALID_ARG;
  if (num_tokens == 0) return GR_OK;
  if (!out || !scale || !x || out_stride < (features + 1) / 2 || x_stride < features || scale_stride < (features + 31) / 32)
    return GR_ERR_INVALID_ARG;
  if (features % 32 != 0 || !aligned(x, 16) || x_stride * dtype_size(dtype) % 16 != 0 || !aligned(out, 16) ||
      out_stride % 16 != 0 || (int64_t)num_tokens * (features / 32) > (1 << 29) - (1 << 20))
    return GR_ERR_UNSUPPORTED;
  const MxQuantArgs a{static_cast<uint8_t*>(out), out_stride, scale, scale_stride, x, x_stride, num_tokens, features};
  const int64_t items = (int64_t)num_tokens * (features / (dtype == GR_DTYPE_F32 ? 8 : 16));
  const dim3 grid((unsigned)((items + MXQ_THREADS - 1) / MXQ_THREADS)), block(MXQ_THREADS);
  auto go = [&](auto k) { hipLaunchKernelGGL(k, grid, block, 0, stream, a); };
  if (dtype == GR_DTYPE_F32) go(mx_quant_k<GR_DTYPE_F32>);
  else if (dtype == GR_DTYPE_F16) go(mx_quant_k<GR_DTYPE_F16>);
  else go(mx_quant_k<GR_DTYPE_BF16>);
  return launch_status();
}

extern "C" gr_status_t gr_dequant_mxfp4(void* out, int64_t out_stride, const void* x, int64_t x_stride,
                                        const uint8_t* scale, int64_t scale_stride, int num_tokens, int features,
                                        int dtype, hipStream_t stream) {
  if (num_tokens < 0 || features < 1 || !dtype_valid(dtype)) return GR_ERR_INVALID_ARG;
  if (num_tokens == 0) return GR_OK;
  if (!out || !scale || !x || out_stride < features || x_stride < (features + 1) / 2 || scale_stride < (features + 31) / 32)
    return GR_ERR_INVALID_ARG;
  if (features % 32 != 0 || !aligned(x, 4) || x_stride % 4 != 0 || !aligned(out, 16) ||
      out_stride * dtype_size(dtype) % 16 != 0 || (int64_t)num_tokens * (features / 32) > (1 << 29) - (1 << 20))
    return GR_ERR_UNSUPPORTED;
  const MxDequantArgs a{out, out_stride, static_cast<const uint8_t*>(x), x_stride, scale, scale_stride, num_tokens, features};
  const int64_t items = ((int64_t)num_tokens + 1) / 2 * (features / 8);
  const dim3 grid((unsigned)((items + MXQ_THREADS - 1) / MXQ_THREADS)), block(MXQ_THREADS);
  auto go = [&](auto k) { hipLaunchKernelGGL(k, grid, block, 0, stream, a); };
  if (dtype == GR_DTYPE_F32) go(mx_dequant_k<GR_DTYPE_F32>);
  else if (dtype == GR_DTYPE_F16) go(mx_dequant_k<GR_DTYPE_F16>);
  else go(mx_dequant_k<GR_DTYPE_BF16>);
  return launch_status();
}

extern "C" int gr_linear_mxfp4_tile(int num_tokens, int out_features, int in_features, int swiglu, int out_dtype) {
  if (num_tokens < 1 || out_features < 1 || in_features < 1 || num_tokens > (1 << 28) || out_features > (1 << 28)) return 0;
  const int i = pick_linear_mx(num_tokens, out_features, in_features / 2, swiglu != 0, out_dtype == GR_DTYPE_MXFP4);
  if (i < 0) return 16 * 1000 - 16 * i * (swiglu ? 2 : 1);
  return 1000000 * kMx[i].per_cu + 1000 * kMx[i].bm + kMx[i].bn;
}

extern "C" gr_status_t gr_linear_mxfp4(void* out, int64_t out_stride, uint8_t* out_scale, int64_t out_scale_stride,
                                       const void* x, int64_t x_stride, const uint8_t* x_scale, int64_t x_scale_stride,
                                       const void* w, int64_t w_stride, const uint8_t* w_scale, int64_t w_scale_stride,
                                       int num_tokens, int out_features, int in_features, int swiglu, int out_dtype,
                                       hipStream_t stream) {
  const bool quant = out_dtype == GR_DTYPE_MXFP4;
  if (num_tokens < 0 || out_features < 1 || in_features < 1 || (swiglu != 0 && swiglu != 1) ||
      (!dtype_valid(out_dtype) && !quant))
    return GR_ERR_INVALID_ARG;
  if (num_tokens == 0) return GR_OK;
  const int64_t row = ((int64_t)in_features + 1) / 2, row_scales = ((int64_t)in_features + 31) / 32;
  if (!out || !x || !x_scale || !w || !w_scale || x_stride < row || w_stride < row || x_scale_stride < row_scales ||
      w_scale_stride < row_scales || out_stride < (quant ? ((int64_t)out_features + 1) / 2 : out_features) ||
      (quant && (!out_scale || out_scale_stride < ((int64_t)out_features + 31) / 32)))
    return GR_ERR_INVALID_ARG;
  if (in_features % 32 != 0 || (swiglu && out_features % 16 != 0) || (quant && out_features % 32 != 0) ||
      out_features > (1 << 28) || num_tokens > (1 << 28) || x_stride > (1 << 22) || w_stride > (1 << 22) ||
      !aligned(x, 16) || x_stride % 16 != 0 || !aligned(w, 16) || w_stride % 16 != 0 ||
      !aligned(out, out_dtype == GR_DTYPE_F32 || quant ? 16 : 8) || (quant && out_stride % 16 != 0) ||
      ((int64_t)num_tokens + 63) / 64 * ((out_features + 63) / 64) > (1 << 23) - 8)
    return GR_ERR_UNSUPPORTED;
  MxArgs a{};
  a.x = static_cast<const uint8_t*>(x);
  a.x_stride = x_stride;
  a.xs4 = x_scale;
  a.xs4_row = x_scale_stride;
  a.w = static_cast<const uint8_t*>(w);
  a.w_stride = w_stride;
  a.ws4 = w_scale;
  a.ws4_row = w_scale_stride;
  a.out = out;
  a.out_stride = out_stride;
  a.os4 = out_scale;
  a.os4_row = out_scale_stride;
  a.M = num_tokens;
  a.N = out_features;
  a.kbytes = in_features / 2;
  a.blocks = in_features / 32;
  a.scale_piece = mx_scale_piece(a);
  a.out_type = out_dtype;
  if (quant) {
    if (swiglu) launch_linear_mx<MM_SWIGLU_Q>(a, stream);
    else launch_linear_mx<MM_PLAIN_Q>(a, stream);
  } else {
    if (swiglu) launch_linear_mx<MM_SWIGLU>(a, stream);
    else launch_linear_mx<MM_PLAIN>(a, stream);
  }
  return launch_status();
}
