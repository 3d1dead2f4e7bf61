/*
 * gr_experts.h -- 8-bit block-scaled projections and routed experts of the
 * decoder that drives the beam path (libgr_beam.so).
 *
 * Same conventions as gr_decoder.h: stream-ordered, no allocation, no host
 * synchronisation, element strides, sums in float32.  An e4m3 tensor
 * (GR_DTYPE_FP8_E4M3) carries float32 scales: one for each 128 features of a
 * row of activations, one for each block of 128 x 128 of a weight matrix (the
 * last of either may be short).  A value is its e4m3 number times its scale.
 */
#ifndef GR_EXPERTS_H_
#define GR_EXPERTS_H_

#include "gr_beam.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Rows to e4m3: for each group of 128 features of a row (the last may be short),
 *   scale = max(float32(max |x| / 448), 2^-80)
 *   out   = the e4m3 number nearest to x / scale, ties to even
 * (of the exact quotient: it is not rounded to float32 in between).  A group with
 * an infinity or a NaN gets that as its scale, so it reads back as NaN where the
 * scale is, or the product of 0 and infinity.  x [num_tokens, features] float32,
 * fp16 or bf16; features % 16 == 0, rows of x and out 16-byte aligned, at most 2^28
 * groups.
 * scale [num_tokens, ceil(features / 128)] at the element strides scale_row /
 * scale_group.
 */
gr_status_t gr_quant_fp8(void* out, int64_t out_stride, float* scale, int64_t scale_row, int64_t scale_group,
                         const void* x, int64_t x_stride, int num_tokens, int features, int dtype,
                         hipStream_t stream);

/*
 * Product of quantised rows and block-scaled weights:
 *   out[t, n] = sum_b x_scale[t, b] * w_scale[n / 128, b] * sum_{k in block b} x[t, k] w[n, k]
 * x [num_tokens, in_features] e4m3 with x_scale at strides x_scale_row /
 * x_scale_group, w [out_features, in_features] e4m3 with w_scale
 * [ceil(out_features / 128), ceil(in_features / 128)] contiguous.
 * swiglu: w is [2 * out_features, in_features] (gate | up), w_scale
 * [2 * ceil(out_features / 128), ...] (gate's blocks, then up's) and
 * out = silu(gate) * up, out_features % 16 == 0.  silu is within
 * 2^-20 + |gate| 2^-23 of itself; a gate below -91.8, where it is no normal float32
 * number, may count as 0.
 * out: out_dtype float32, fp16 or bf16, rounded once; or GR_DTYPE_FP8_E4M3: the
 * float32 results quantised as gr_quant_fp8 does, with out_scale at strides
 * out_scale_row / out_scale_group (needs out_features % 16 == 0).  out is 16-byte
 * aligned for float32 and 8-byte for 16 bits, at any row stride; e4m3 rows are each
 * 4-byte aligned.
 * Sums are float32 throughout for a float32 or e4m3 result.  For a 16-bit one the
 * matrix core adds the e4m3 products, in groups of 8 whose members are cut off
 * below 2^-13 of the largest (about 1.5e-5 of an ordinary result); the groups'
 * sums are float32.  The sizes of a call choose its kernel, and with it the order
 * of the sums and, for small results, float32 sums of 16-bit ones too: a row's last
 * bits may differ between calls of other sizes (not between calls of the same).
 * x_scale * w_scale is formed first, in float32: a block where that overflows is
 * infinite or NaN, one where it is below 2^-126 keeps as many bits as that has.
 * in_features % 16 == 0; x and w rows 16-byte aligned, at most 4 MB apart; no more
 * than 2^35 results, less for sizes that leave 64 x 64 tiles part empty.
 */
gr_status_t gr_linear_fp8(void* out, int64_t out_stride, float* out_scale, int64_t out_scale_row,
                          int64_t out_scale_group, const void* x, int64_t x_stride, const float* x_scale,
                          int64_t x_scale_row, int64_t x_scale_group, const void* w, int64_t w_stride,
                          const float* w_scale, int num_tokens, int out_features, int in_features, int swiglu,
                          int out_dtype, hipStream_t stream);

enum { GR_SCORE_SOFTMAX = 0, GR_SCORE_SIGMOID = 1 };

/*
 * Experts of each token from its router logits [num_tokens, num_experts]:
 *   s = softmax(logits) or sigmoid(logits);  c = s + bias, or the logits without a bias
 * With num_groups > 1 the experts are that many equal runs; a group's value is the
 * sum of its two largest c (its largest without a bias) and only experts of the
 * top_groups best groups are considered.  ids[t] = the top_k considered experts by
 * c, largest first; weights[t, j] = scale * s[ids[t, j]], divided by the chosen
 * ones' sum if renormalize (a sum of 0 gives weights of 0).  Ties, of c and of
 * groups' values, go to the lowest index.  c and the groups' values are compared
 * as computed in float64.  A row of -inf alone has s = 0; a NaN ranks last.
 * logits float32, fp16 or bf16 at logits_stride, bias float32 [num_experts] or
 * NULL; weights float32, ids int32 [num_tokens, top_k] contiguous.
 * num_experts <= 1024, num_groups <= 64, top_k <= 64, at most 2^34 logits.
 */
gr_status_t gr_route_experts(float* weights, int32_t* ids, const void* logits, int64_t logits_stride,
                             const float* bias, int num_tokens, int num_experts, int top_k, int score,
                             int num_groups, int top_groups, int renormalize, float scale, int dtype,
                             hipStream_t stream);

/*
 * SwiGLU layers of the chosen experts:
 *   out[t] = sum_j weights[t, j] * down[e] (silu(gate[e] x[t]) * (up[e] x[t])),  e = ids[t, j]
 * x, out [num_tokens, hidden] fp16 or bf16 at their strides; gate_up
 * [num_experts, 2 * ffn, hidden] (gate | up) and down [num_experts, hidden, ffn]
 * contiguous; weights float32, ids int32 [num_tokens, top_k] contiguous.  An id
 * below 0 adds nothing (an expert of another rank), one >= num_experts flags
 * GR_DEV_BAD_EXPERT and adds nothing; an expert named twice counts twice.
 * Without scales the weights are of x's type, and the gated product of each
 * expert is rounded to it.  With gate_up_scale [num_experts, 2 * ceil(ffn / 128),
 * ceil(hidden / 128)] and down_scale [num_experts, ceil(hidden / 128),
 * ceil(ffn / 128)] they are e4m3, and x and the gated products are quantised as
 * gr_quant_fp8 does.  Sums are float32 (of e4m3 weights in the down product as for
 * gr_linear_fp8's 16-bit results), and with e4m3 weights or a bf16 out each expert's
 * result is rounded to fp16 times a power of two (2^-11 of a value, 2^-39 of the
 * largest of its 16 to 64 neighbouring columns) before the sum over j, which is
 * float32 and in the order of j.  As for gr_linear_fp8, a token's last bits may
 * differ between calls of other sizes.
 * hidden % 16 == 0, ffn % 16 == 0; rows of x, and weights, 16-byte aligned; out
 * rows 8-byte aligned.  num_experts <= 1024, num_tokens < 2^23, x spans less than
 * 2 GB.  workspace: gr_expert_mlp_workspace_size bytes, 256-byte aligned, no initial
 * contents; calls that may overlap need one each.
 */
size_t gr_expert_mlp_workspace_size(int num_tokens, int top_k, int num_experts, int hidden, int ffn, int fp8);
gr_status_t gr_expert_mlp(void* out, int64_t out_stride, const void* x, int64_t x_stride, const void* gate_up,
                          const float* gate_up_scale, const void* down, const float* down_scale,
                          const float* weights, const int32_t* ids, int num_tokens, int top_k, int num_experts,
                          int hidden, int ffn, int dtype, void* workspace, size_t workspace_bytes,
                          int32_t* dev_status, hipStream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* GR_EXPERTS_H_ */
