// Activations to e4m3 in groups of 128, and the product of such rows with
// weights that have a scale for each block of 128 x 128 (gr_block_mm.h).
#include "gr_block_mm.h"

namespace gr {
namespace {

constexpr int QT_THREADS = 256, QT_GROUPS = QT_THREADS / 8;

template <int DT, int ROWS> __global__ __launch_bounds__(QT_THREADS) void quant_fp8_k(QuantArgs a) {
  // (items: below 2^31 by the entry's check)
  quant_group<DT, ROWS>(a, blockIdx.x * QT_GROUPS + (threadIdx.x >> 3), threadIdx.x & 7);
}

// The tile with the least estimated time, over the workgroups of the XCD that gets
// the most of them (its 32 CUs take one or two each): a round costs a fixed part
// (launch, first stages, stores) and its stages, `one` ns each alone on a CU, `two`
// with a neighbour.  From 512 to 12288 columns and 64 to 2048 rows of 2048 and 6144
// features (weights cold; measured, us, the picked tile's and the next best one's):
//   64 x 4096 (2048 in)   64 x 64    8.5,  64 x 128 10.3
//   512 x 8192            64 x 128  17.5, 128 x 128 18.5
//   1000 x 12288         256 x 256  33.9, 128 x 128 39.9
//   2048 x 12288         256 x 256  67.4, 128 x 128 63.7  (the estimate is within 6 %)
//   1000 x 2048 (6144 in) 64 x 128  27.4,  64 x 64  30.0
// A float32 result's stages convert their operands and take longer; 256 x 256 has no
// registers for that.
struct MmChoice { int bm, bn, per_cu, fixed, one, two; };
constexpr MmChoice kFast[] = {{64, 64, 2, 2300, 400, 570}, {64, 128, 2, 2500, 510, 820}, {128, 128, 2, 1500, 900, 1260},
                              {128, 256, 1, 2000, 1100, 0}, {256, 256, 1, 4000, 1600, 0}};
constexpr MmChoice kExact[] = {{64, 64, 2, 2300, 500, 860}, {64, 128, 2, 2500, 750, 1310}, {128, 128, 2, 1500, 1150, 2000},
                               {128, 256, 1, 2000, 1750, 0}};

template <int N> int pick_tile(const MmChoice (&all)[N], int M, int rows_w, int stages) {
  int best = 0;
  int64_t least = INT64_MAX;
  for (int i = 0; i < N; ++i) {
    const MmChoice& c = all[i];
    const int64_t tiles = ((int64_t)((M + c.bm - 1) / c.bm) * ((rows_w + c.bn - 1) / c.bn) + 7) / 8;
    const int64_t one = c.fixed + (int64_t)stages * c.one, two = c.fixed + (int64_t)stages * c.two;
    const int64_t round = 32 * c.per_cu, left = tiles % round;
    const int64_t cost = tiles / round * (c.per_cu == 2 ? two : one) + (left == 0 ? 0 : left <= 32 ? one : two);
    if (cost < least) {
      least = cost;
      best = i;
    }
  }
  return best;
}

template <int MODE, bool EXACT>
void launch_linear_fp8(const MmArgs& a, hipStream_t stream) {
  constexpr int T = GR_DTYPE_FP8_E4M3;
  constexpr bool GATED = MODE == MM_SWIGLU || MODE == MM_SWIGLU_Q;
  const int M = a.M, rows_w = GATED ? 2 * a.N : a.N, stages = (a.kbytes + 127) / 128;
  if constexpr (MODE == MM_PLAIN_Q) {
    launch_mm<T, 64, 128, 2, 4, 3, MODE, false, EXACT>(a, (M + 63) / 64, stream);
  } else if constexpr (MODE == MM_SWIGLU_Q) {
    // a group of 128 results is 256 weight rows of one workgroup, which leaves little choice
    const int64_t cols = (a.N + 127) / 128;
    if ((M + 63) / 64 * cols <= 256) launch_mm<T, 64, 256, 2, 4, 3, MODE, false, EXACT>(a, (M + 63) / 64, stream);
    else launch_mm<T, 128, 256, 2, 4, 3, MODE, false, EXACT>(a, (M + 127) / 128, stream);
  } else {
    // as long as two workgroups a CU hold them all (8 rows x 4096 columns 4.8 us, by 64 x 64 tiles 8.7; 64 x 4096
    // 8.5; 64 x 8192, twice that many, 14.5 against 9.5)
    const int64_t cols = (a.N + 15) / 16, few = (M + 15) / 16 * cols, few2 = (M + 31) / 32 * cols;
    if (few <= 256 || (M <= 16 && few <= 512)) return launch_few<T, 1, MODE, false>(a, (M + 15) / 16, stream);
    if (few2 <= 512) return launch_few<T, 2, MODE, false>(a, (M + 31) / 32, stream);
    switch (EXACT ? pick_tile(kExact, M, rows_w, stages) : pick_tile(kFast, M, rows_w, stages)) {
      case 0: launch_mm<T, 64, 64, 2, 2, 4, MODE, false, EXACT>(a, (M + 63) / 64, stream); break;
      case 1: launch_mm<T, 64, 128, 2, 2, 3, MODE, false, EXACT>(a, (M + 63) / 64, stream); break;
      case 2: launch_mm<T, 128, 128, 2, 2, 2, MODE, false, EXACT>(a, (M + 127) / 128, stream); break;
      case 3: launch_mm<T, 128, 256, 2, 4, 3, MODE, false, EXACT>(a, (M + 127) / 128, stream); break;
      default:
        if constexpr (!EXACT) launch_mm<T, 256, 256, 2, 4, 2, MODE, false, EXACT>(a, (M + 255) / 256, stream);
    }
  }
}

}  // namespace

}  // namespace gr

using namespace gr;

namespace {
bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
}  // namespace

extern "C" gr_status_t gr_quant_fp8(void* out, int64_t out_stride, float* scale, int64_t scale_row,
                                    int64_t scale_group, const void* x, int64_t x_stride, int num_tokens,
                                    int features, int dtype, hipStream_t stream) {
  if (num_tokens < 0 || features < 1 || !dtype_valid(dtype)) return GR_ERR_INVALID_ARG;
  if (num_tokens == 0) return GR_OK;
  if (!out || !scale || !x || out_stride < features || x_stride < features || scale_row < 0 || scale_group < 0)
    return GR_ERR_INVALID_ARG;
  if (features % 16 != 0 || !aligned(x, 16) || x_stride * dtype_size(dtype) % 16 != 0 || !aligned(out, 16) ||
      out_stride % 16 != 0 || !aligned(scale, 4) || (int64_t)num_tokens * ((features + 127) / 128) > (1 << 28))
    return GR_ERR_UNSUPPORTED;
  const QuantArgs a{static_cast<uint8_t*>(out), out_stride, scale, scale_row, scale_group, x, x_stride,
                    num_tokens, features, (features + 127) / 128};
  const int rows = quant_rows(num_tokens, a.groups);
  const int64_t items = ((int64_t)num_tokens + rows - 1) / rows * a.groups;
  const dim3 grid((unsigned)((items + QT_GROUPS - 1) / QT_GROUPS)), block(QT_THREADS);
  auto go = [&](auto one, auto two) { hipLaunchKernelGGL(rows == 2 ? two : one, grid, block, 0, stream, a); };
  if (dtype == GR_DTYPE_F32) go(quant_fp8_k<GR_DTYPE_F32, 1>, quant_fp8_k<GR_DTYPE_F32, 2>);
  else if (dtype == GR_DTYPE_F16) go(quant_fp8_k<GR_DTYPE_F16, 1>, quant_fp8_k<GR_DTYPE_F16, 2>);
  else go(quant_fp8_k<GR_DTYPE_BF16, 1>, quant_fp8_k<GR_DTYPE_BF16, 2>);
  return launch_status();
}

extern "C" gr_status_t gr_linear_fp8(void* out, int64_t out_stride, float* out_scale, int64_t out_scale_row,
                                     int64_t out_scale_group, const void* x, int64_t x_stride, const float* x_scale,
                                     int64_t x_scale_row, int64_t x_scale_group, const void* w, int64_t w_stride,
                                     const float* w_scale, int num_tokens, int out_features, int in_features,
                                     int swiglu, int out_dtype, hipStream_t stream) {
  const bool quant = out_dtype == GR_DTYPE_FP8_E4M3;
  if (num_tokens < 0 || out_features < 1 || in_features < 1 || (swiglu != 0 && swiglu != 1) ||
      (!dtype_valid(out_dtype) && !quant))
    return GR_ERR_INVALID_ARG;
  if (num_tokens == 0) return GR_OK;
  if (!out || !x || !x_scale || !w || !w_scale || out_stride < out_features || x_stride < in_features ||
      w_stride < in_features || x_scale_row < 0 || x_scale_group < 0 ||
      (quant && (!out_scale || out_scale_row < 0 || out_scale_group < 0)))
    return GR_ERR_INVALID_ARG;
  if (in_features % 16 != 0 || ((swiglu || quant) && out_features % 16 != 0) || out_features > (1 << 28) ||
      num_tokens > (1 << 28) || x_stride > (1 << 22) || w_stride > (1 << 22) || !aligned(x, 16) || x_stride % 16 != 0 ||
      !aligned(w, 16) || w_stride % 16 != 0 ||
      !aligned(out, out_dtype == GR_DTYPE_F32 ? 16 : quant ? 4 : 8) || (quant && out_stride % 4 != 0) ||
      !aligned(x_scale, 4) || !aligned(w_scale, 4) || (quant && !aligned(out_scale, 4)) ||
      x_scale_group > INT32_MAX || ((int64_t)num_tokens + 63) / 64 * ((out_features + 63) / 64) > (1 << 23) - 8)
    return GR_ERR_UNSUPPORTED;
  MmArgs a{};
  a.x = static_cast<const uint8_t*>(x);
  a.x_stride = x_stride;
  a.xs = x_scale;
  a.xs_row = x_scale_row;
  a.xs_grp = x_scale_group;
  a.w = static_cast<const uint8_t*>(w);
  a.w_stride = w_stride;
  a.ws = w_scale;
  a.out = out;
  a.out_stride = out_stride;
  a.out_scale = out_scale;
  a.os_row = out_scale_row;
  a.os_grp = out_scale_group;
  a.M = num_tokens;
  a.N = out_features;
  a.kbytes = in_features;
  a.out_type = out_dtype;
  if (quant) {
    if (swiglu) launch_linear_fp8<MM_SWIGLU_Q, true>(a, stream);
    else launch_linear_fp8<MM_PLAIN_Q, true>(a, stream);
  } else if (out_dtype == GR_DTYPE_F32) {
    if (swiglu) launch_linear_fp8<MM_SWIGLU, true>(a, stream);
    else launch_linear_fp8<MM_PLAIN, true>(a, stream);
  } else {
    if (swiglu) launch_linear_fp8<MM_SWIGLU, false>(a, stream);
    else launch_linear_fp8<MM_PLAIN, false>(a, stream);
  }
  return launch_status();
}
