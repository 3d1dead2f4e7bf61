/*
 * gr_mxfp4.h -- 4-bit microscaled (MXFP4) activations, projections and routed
 * experts of the decoder that drives the beam path (libgr_beam.so).
 *
 * Same conventions as gr_experts.h: stream-ordered, no allocation, no host
 * synchronisation, sums in float32.  In a 4-bit tensor each 32 neighbouring
 * features of a row share a scale byte, 2^(byte - 127) (255: NaN), and a number is
 * one of e2m1's 0, 0.5, 1, 1.5, 2, 3, 4, 6 (codes 0 to 7; 8 to 15 their negatives).
 * Two codes a byte, the even feature's in the low four bits: a row of K features is
 * K / 2 bytes and K / 32 scale bytes, K a multiple of 32.  Strides of 4-bit rows and
 * of scale rows are in bytes, the scale bytes of a row lie side by side.
 */
#ifndef GR_MXFP4_H_
#define GR_MXFP4_H_

#include "gr_beam.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { GR_DTYPE_MXFP4 = 4 }; /* an output of gr_linear_mxfp4 */

/*
 * Rows to 4 bits.  A block's scale is the smallest 2^e, e >= -127, with
 * max |x| < 7 * 2^e (at which its largest rounds to 6 at most); its numbers are the
 * e2m1 ones nearest to x / 2^e, ties to the even code, with x's sign.  A block with
 * an infinity or a NaN gets the scale byte 255 and reads back as NaN.
 * x [num_tokens, features] float32, fp16 or bf16 at x_stride elements; rows of x and
 * out 16-byte aligned; fewer than 2^29 - 2^20 blocks.
 */
gr_status_t gr_quant_mxfp4(void* out, int64_t out_stride, uint8_t* scale, int64_t scale_stride, const void* x,
                           int64_t x_stride, int num_tokens, int features, int dtype, hipStream_t stream);

/*
 * And back: out[t, k] = round(number * scale) as float32, fp16 or bf16.  Rows of x
 * 4-byte aligned, rows of out 16-byte aligned; as many blocks as above.
 */
gr_status_t gr_dequant_mxfp4(void* out, int64_t out_stride, const void* x, int64_t x_stride, const uint8_t* scale,
                             int64_t scale_stride, int num_tokens, int features, int dtype, hipStream_t stream);

/*
 * Product of 4-bit rows and 4-bit weights:
 *   out[t, n] = sum_b x_scale[t, b] * w_scale[n, b] * sum_{k in block b} x[t, k] w[n, k]
 * x [num_tokens, in_features], w [out_features, in_features].
 * swiglu: w is [2 * out_features, in_features] (gate | up) and out = silu(gate) * up,
 * out_features % 16 == 0; silu as for gr_linear_fp8.
 * out: out_dtype float32, fp16 or bf16, rounded once (16-byte aligned for float32,
 * 8-byte for 16 bits, at any row stride); or GR_DTYPE_MXFP4: the float32 results in
 * 4 bits as gr_quant_mxfp4 has them, with out_scale (rows of out 16-byte aligned,
 * out_features % 32 == 0).
 * Sums are float32: a block's 32 products are added exactly, four blocks are joined
 * within 2^-24 of their sum of magnitudes.  A pair of scales whose product is above
 * 2^127 or below 2^-126 gives infinities or flushed results as float32 does.  The
 * sizes of a call choose its kernel, and with it the order of the sums: a row's float32
 * sums may differ in their last bits between calls of other sizes (not between calls of
 * the same).  In a 4-bit result such a difference can take a number that lies at a
 * border to the next one, and a block whose largest lies at one to the next scale, by
 * which all its numbers are rounded: what is made of it then depends on the number of
 * rows in the call by as much as the format resolves.
 * in_features % 32 == 0; x and w rows 16-byte aligned, at most 4 MB apart;
 * num_tokens and out_features <= 2^28, no more than 2^35 results, less for sizes that
 * leave 64 x 64 tiles part empty.
 */
gr_status_t gr_linear_mxfp4(void* out, int64_t out_stride, uint8_t* out_scale, int64_t out_scale_stride, const void* x,
                            int64_t x_stride, const uint8_t* x_scale, int64_t x_scale_stride, const void* w,
                            int64_t w_stride, const uint8_t* w_scale, int64_t w_scale_stride, int num_tokens,
                            int out_features, int in_features, int swiglu, int out_dtype, hipStream_t stream);

/*
 * The tile that gr_linear_mxfp4 takes for these sizes: 1000 * rows + weight rows, with
 * 1000000 * the tiles that share a CU (0: the few rows' kernel, of 16 rows); 0 for
 * sizes that are not positive or above 2^28.
 */
int gr_linear_mxfp4_tile(int num_tokens, int out_features, int in_features, int swiglu, int out_dtype);

/*
 * SwiGLU layers of the chosen experts with 4-bit weights:
 *   out[t] = sum_j weights[t, j] * down[e] q(silu(gate[e] q(x[t])) * (up[e] q(x[t]))),  e = ids[t, j]
 * with q as gr_quant_mxfp4.  x, out [num_tokens, hidden] fp16 or bf16 at their strides
 * (elements); gate_up [num_experts, 2 * ffn, hidden] (gate | up) and down [num_experts,
 * hidden, ffn] with their scales, all contiguous; weights float32, ids int32
 * [num_tokens, top_k] contiguous.  An id below 0 adds nothing (an expert of another
 * rank), one >= num_experts flags GR_DEV_BAD_EXPERT and adds nothing; an expert named
 * twice counts twice.  Sums are float32, the one over j too, which is in the order of j
 * and rounded once.  A token's result depends on its own row, choices and the experts
 * alone: it has the same bits whatever other tokens the call has.
 * hidden % 32 == 0, ffn % 32 == 0; rows of x, and weights, 16-byte aligned; out rows
 * 8-byte aligned.  num_experts <= 1024, hidden and ffn <= 2^21, num_tokens < 2^23,
 * num_tokens * top_k <= 2^26, num_tokens * hidden <= 2^32 - 2^24, and fewer than 2^23 - 8
 * workgroups: num_tokens * top_k over a tile's rows, plus one for each expert, times the
 * larger of hidden and ffn over 64 (128 for tiles of 128 and 256 rows).
 * workspace: gr_expert_mlp_mxfp4_workspace_size bytes, 256-byte aligned, no initial
 * contents; one for more tokens does for fewer; calls that may overlap need one each.
 */
size_t gr_expert_mlp_mxfp4_workspace_size(int num_tokens, int top_k, int num_experts, int hidden, int ffn);
gr_status_t gr_expert_mlp_mxfp4(void* out, int64_t out_stride, const void* x, int64_t x_stride, const void* gate_up,
                                const uint8_t* gate_up_scale, const void* down, const uint8_t* down_scale,
                                const float* weights, const int32_t* ids, int num_tokens, int top_k, int num_experts,
                                int hidden, int ffn, int dtype, void* workspace, size_t workspace_bytes,
                                int32_t* dev_status, hipStream_t stream);

/*
 * The tiles that gr_expert_mlp_mxfp4 takes for these sizes: 1000000 * stages of the gated
 * product on their way + 1000 * rows + columns of the down product; 0 for sizes that
 * are not positive, and for features above 2^21.
 */
int gr_expert_mlp_mxfp4_tile(int num_tokens, int top_k, int num_experts, int hidden, int ffn);

#ifdef __cplusplus
}
#endif
#endif /* GR_MXFP4_H_ */
