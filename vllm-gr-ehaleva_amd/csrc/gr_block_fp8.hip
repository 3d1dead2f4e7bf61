// Activations to e4m3 in groups of 128, and the product of such rows with
// weights that have a scale for each block of 128 x 128 (gr_block_mm.h).
#include "gr_block_mm.h"

namespace gr {
namespace {

constexpr int QT_THREADS = 256;

struct QuantArgs {
  uint8_t* out;
  int64_t out_stride;
  float* scale;
  int64_t scale_row, scale_grp;
  const void* x;
  int64_t x_stride;
  int T, K, groups;
};

// One group of 128 features per 16 lanes, 8 features a lane; a workgroup's 16
// groups are neighbours in their row.
template <int DT>
__global__ __launch_bounds__(QT_THREADS) void quant_fp8_k(QuantArgs a) {
  using E = Elem<DT>;
  using S = typename E::storage;
  struct alignas(16) Vec { S e[8]; };
  const int64_t item = (int64_t)blockIdx.x * (QT_THREADS / 16) + (threadIdx.x >> 4);
  const int l = threadIdx.x & 15;
  const int64_t t = item / a.groups;
  const int g = (int)(item - t * a.groups);
  if (t >= a.T) return;  // whole 16-lane groups leave together
  const int k = g * 128 + l * 8;
  float v[8] = {};
  uint32_t m = 0;
  if (k < a.K) {
    const Vec in = *reinterpret_cast<const Vec*>(static_cast<const S*>(a.x) + t * a.x_stride + k);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = E::to_float(in.e[i]);
      m = max(m, __builtin_bit_cast(uint32_t, v[i]) & 0x7FFFFFFFu);
    }
  }
#pragma unroll
  for (int off = 8; off > 0; off >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, off, 16));
  const float s = quant_scale(m), r = 1.0f / s;
  if (k < a.K) {
    const float lo[4] = {v[0], v[1], v[2], v[3]}, hi[4] = {v[4], v[5], v[6], v[7]};
    *reinterpret_cast<u32x2_t*>(a.out + t * a.out_stride + k) = u32x2_t{quant_pack4(lo, s, r), quant_pack4(hi, s, r)};
  }
  if (l == 0) a.scale[t * a.scale_row + g * a.scale_grp] = s;
}

template <int MODE, bool EXACT>
void launch_linear_fp8(const MmArgs& a, hipStream_t stream) {
  constexpr int BN = MODE == MM_PLAIN_Q ? 128 : 256;
  launch_mm<GR_DTYPE_FP8_E4M3, 64, BN, 2, 4, 3, MODE, false, EXACT>(a, (a.M + 63) / 64, stream);
}

}  // namespace

gr_status_t launch_quant_fp8(void* out, int64_t out_stride, float* scale, int64_t scale_row, int64_t scale_group,
                             const void* x, int64_t x_stride, int num_tokens, int features, int dtype,
                             hipStream_t stream) {
  QuantArgs a{static_cast<uint8_t*>(out), out_stride, scale, scale_row, scale_group, x, x_stride,
              num_tokens, features, (features + 127) / 128};
  const int64_t items = (int64_t)num_tokens * a.groups, per = QT_THREADS / 16;
  const dim3 grid((unsigned)((items + per - 1) / per)), block(QT_THREADS);
  if (dtype == GR_DTYPE_F32) hipLaunchKernelGGL(quant_fp8_k<GR_DTYPE_F32>, grid, block, 0, stream, a);
  else if (dtype == GR_DTYPE_F16) hipLaunchKernelGGL(quant_fp8_k<GR_DTYPE_F16>, grid, block, 0, stream, a);
  else hipLaunchKernelGGL(quant_fp8_k<GR_DTYPE_BF16>, grid, block, 0, stream, a);
  return launch_status();
}

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
  if (features % 16 != 0 || !aligned(x, 16) || x_stride * dtype_size(dtype) % 16 != 0 || !aligned(out, 8) ||
      out_stride % 8 != 0 || !aligned(scale, 4) || (int64_t)num_tokens * ((features + 127) / 128) > INT32_MAX)
    return GR_ERR_UNSUPPORTED;
  return launch_quant_fp8(out, out_stride, scale, scale_row, scale_group, x, x_stride, num_tokens, features, dtype,
                          stream);
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
      num_tokens > (1 << 28) || !aligned(x, 16) || x_stride % 16 != 0 || !aligned(w, 16) || w_stride % 16 != 0 ||
      !aligned(out, out_dtype == GR_DTYPE_F32 ? 16 : quant ? 4 : 8) || (quant && out_stride % 4 != 0) ||
      !aligned(x_scale, 4) || !aligned(w_scale, 4) || (quant && !aligned(out_scale, 4)) ||
      ((int64_t)num_tokens + 15) / 16 * ((out_features + 15) / 16) > INT32_MAX - 8)
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
