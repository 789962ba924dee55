/*
 * mdlayers.h -- C ABI of the layers beside attention in a DiT block: layer norm and RMS norm with their backward passes, quantisation to
 * e4m3 in blocks of 128, and the product of such operands.
 *
 * Part of libmdattn.so, with the conventions and the MDATTN_E_* codes of mdattn.h: a HIP stream first, work only enqueued,
 * nothing allocated or synchronised, arguments checked on the host before any launch, caller-owned device pointers,
 * re-entrant.
 *
 * A grid has fewer than 2^32 threads: MDATTN_E_UNSUPPORTED, before anything is launched, for norms of more than 2^32 / 1024 groups that
 * are not walked as one and need more, for dw and db of more than 2^22 groups x 64 channels, and for quantising 2^38 elements.
 */
#ifndef MDLAYERS_H_
#define MDLAYERS_H_

#include "mdattn.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Layer norm of rows of C channels:  y = h * (w_offset + w) + b,  h = (x - mean) / sqrt(var + eps).
 * Replaces FP32LayerNorm with adaLN's scale and shift (w_offset 1, w and b per batch element; models/wan/transformers/
 * transformer_wan.py:487) and the affine norm of the cross-attention (w_offset 0, w and b shared).
 *   x, y          bf16 or f32 (x_is_f32, y_is_f32), [groups, rows, C] by the strides of a group and of a row, in elements;
 *                 C contiguous.  A group is what shares w and b: a batch element.  y may be x where types and strides agree.
 *   w, b          bf16 or f32 (wb_is_f32), C channels each, dense; wb_stride elements between groups, 0: shared.  Either may be
 *                 NULL: y = h + b whatever w_offset is, y = h * (w_offset + w).
 * Statistics and arithmetic in f32, the variance from differences to the mean, one rounding.
 * 1 <= C <= 16384; pointers and strides need the alignment of an element only.
 */
int mdattn_layer_norm(void* stream, const void* x, int x_is_f32, void* y, int y_is_f32, const void* w, const void* b, int wb_is_f32,
                      int64_t groups, int64_t rows, int C, int64_t x_stride_group, int64_t x_stride_row, int64_t y_stride_group,
                      int64_t y_stride_row, int64_t wb_stride, float eps, float w_offset);

/*
 * The same, its output quantised without being stored: q and scales as mdattn_quant_block_e4m3 makes them (block_rows 1) of the
 * unrounded f32 rows, groups * rows of them, dense.
 */
int mdattn_layer_norm_e4m3(void* stream, const void* x, int x_is_f32, void* q, void* scales, const void* w, const void* b, int wb_is_f32,
                           int64_t groups, int64_t rows, int C, int64_t x_stride_group, int64_t x_stride_row, int64_t wb_stride, float eps,
                           float w_offset);

/*
 * Backward of mdattn_layer_norm.  With a = g * (w_offset + w):
 *   dx = (a - mean(a) - h * mean(a h)) / sqrt(var + eps),  dw = sum of g h,  db = sum of g, over the rows that share w and b.
 *   x             the forward's input; its mean and variance are computed again
 *   g             gradient of y, of x's type, by strides of its own; dx of x's type, by its strides
 *   dw, db        of w's type (wb_is_f32), dense, [groups, C] with wb_stride != 0, [C] with 0; either may be NULL
 *   w             may be NULL (then dw has to be NULL too)
 *   workspace     mdattn_layer_norm_bwd_workspace_floats floats; unused, and may be NULL, without dw and db
 * Deterministic: the sums over the rows are made in a fixed order.
 */
int64_t mdattn_layer_norm_bwd_workspace_floats(int64_t groups, int64_t rows, int C);
int mdattn_layer_norm_bwd(void* stream, const void* x, int x_is_f32, const void* g, void* dx, const void* w, void* dw, void* db, int wb_is_f32,
                          int64_t groups, int64_t rows, int C, int64_t x_stride_group, int64_t x_stride_row, int64_t g_stride_group,
                          int64_t g_stride_row, int64_t dx_stride_group, int64_t dx_stride_row, int64_t wb_stride, float eps,
                          float w_offset, float* workspace, int64_t workspace_floats);

/*
 * RMS norm of the sum of x and a residual:  s = x + residual,  y = s * r * (w_offset + w) + b,  r = (mean of s^2 over the row + eps)^-1/2.
 * A prompt encoder's norms (models/qwen3_flax.py), LTX-2's with scale and shift (w_offset 1, w and b per batch element;
 * models/ltx2/transformer_ltx2.py), the addition in front of them done on the way.
 *   x, y          bf16 or f32 (x_is_f32), as mdattn_layer_norm's x
 *   residual      or NULL: s = x; of x's type, or f32 beside a bf16 x (r_is_f32); its own strides.  s, of the residual's type, gets the sum;
 *                 both or neither.  s may be residual, and y x, where the strides agree.
 *   w, b          as mdattn_layer_norm's
 * The norm is that of the unrounded f32 sum.  Arithmetic in f32, one rounding of y and one of s.  1 <= C <= 16384.
 */
int mdattn_rms_norm(void* stream, const void* x, int x_is_f32, const void* residual, int r_is_f32, void* y, void* s, const void* w, const void* b,
                    int wb_is_f32, int64_t groups, int64_t rows, int C, int64_t x_stride_group, int64_t x_stride_row, int64_t r_stride_group,
                    int64_t r_stride_row, int64_t y_stride_group, int64_t y_stride_row, int64_t s_stride_group, int64_t s_stride_row,
                    int64_t wb_stride, float eps, float w_offset);
/* The same, y quantised without being stored: q and scales as mdattn_layer_norm_e4m3 has them. */
int mdattn_rms_norm_e4m3(void* stream, const void* x, int x_is_f32, const void* residual, int r_is_f32, void* q, void* scales, void* s, const void* w,
                         const void* b, int wb_is_f32, int64_t groups, int64_t rows, int C, int64_t x_stride_group, int64_t x_stride_row,
                         int64_t r_stride_group, int64_t r_stride_row, int64_t s_stride_group, int64_t s_stride_row, int64_t wb_stride, float eps,
                         float w_offset);

/*
 * Backward of mdattn_rms_norm.  With a = g * (w_offset + w) and h = s r:
 *   ds = r (a - h mean(a h)) + gs,  dw = sum of g h,  db = sum of g, over the rows that share w and b; x's gradient and the residual's are ds.
 *   s             the forward's sum (x, where it had no residual), bf16 or f32; r is computed again
 *   residual      or NULL; beside an s in bf16 only: s is x, in bf16, to which it is added again, for gradients without s's rounding (dw in f32); its
 *                 own strides
 *   g             gradient of y, bf16 or f32; of s's type, or bf16 beside an f32 s
 *   gs            gradient of s, of its type, or NULL
 *   ds            of s's type;  dx: the same rounded to bf16, where g is bf16 and s f32, or NULL
 *   dw, db        of w's type (wb_is_f32; db has it without w too), as mdattn_layer_norm_bwd's; either may be NULL
 *   workspace     mdattn_rms_norm_bwd_workspace_floats floats; unused, and may be NULL, without dw and db
 * ds and dx are dense [groups, rows, C].  Deterministic.
 */
int64_t mdattn_rms_norm_bwd_workspace_floats(int64_t groups, int64_t rows, int C);
int mdattn_rms_norm_bwd(void* stream, const void* s, int s_is_f32, const void* residual, const void* g, int g_is_f32, const void* gs, void* ds,
                        void* dx, const void* w, void* dw, void* db, int wb_is_f32, int64_t groups, int64_t rows, int C, int64_t s_stride_group,
                        int64_t s_stride_row, int64_t r_stride_group, int64_t r_stride_row, int64_t g_stride_group, int64_t g_stride_row,
                        int64_t gs_stride_group, int64_t gs_stride_row, int64_t wb_stride, float eps, float w_offset, float* workspace,
                        int64_t workspace_floats);

/*
 * Quantisation of x [R, C] to e4m3 with one power-of-two scale per block of block_rows x 128 (block_rows 1 or 128).  Over a block,
 * m = max |x|, e the smallest integer >= -127 with m <= 448 * 2^e; stored are x * 2^-e (round to nearest even) and the byte e + 127
 * (0xFF, a NaN, and NaNs for the values, where the block holds an infinity or a NaN).
 *   x             bf16 or f32, rows x_stride elements apart, C contiguous
 *   q, scales     or NULL: e4m3 bytes [R, ceil128(C)], and [ceil(R / block_rows), ceil4(ceil(C / 128))] scale bytes; dense.  The
 *                 padding of q's rows is zero (NaN in a block that is not finite), that of the scales' rows unspecified.
 *   qt, scales_t  or NULL: the same of x transposed, [C, ceil128(R)], blocks of block_rows x 128 of the transposed matrix
 *   colsum        or NULL: f32 [ceil(R / 128), C], the sum of each column over each 128 rows
 * q, qt 16-byte aligned, scales 4-byte aligned; x the alignment of an element.
 */
int mdattn_quant_block_e4m3(void* stream, const void* x, int x_is_f32, int64_t R, int64_t C, int64_t x_stride, int block_rows, void* q,
                            void* scales, void* qt, void* scales_t, float* colsum);
/* out [C] = the sum of the `n` rows of colsum [n, C] (f32 or, out_is_f32 0, bf16), in a fixed order. */
int mdattn_sum_rows(void* stream, const float* rows, int64_t n, int64_t C, void* out, int out_is_f32);

/*
 * c [M, N] (bf16) = a b^T + bias:  a [M, K] with block_rows 1, b [N, K] with block_rows 1 or 128 (b_block_rows), both as
 * mdattn_quant_block_e4m3 stores them; bias bf16 or f32 (bias_is_f32) [N], or NULL.  c's rows are c_stride elements apart.
 * f32 sums on the matrix cores, whose 8-bit forms add eight products at a time with 14 bits below the largest; one rounding.
 *   workspace     mdattn_matmul_fp8_block_workspace_floats floats (0 for most sizes), with which a product of few output tiles is
 *                 split over K; with less it runs unsplit.  16-byte aligned.
 */
int64_t mdattn_matmul_fp8_block_workspace_floats(int64_t M, int64_t N, int64_t K);
int mdattn_matmul_fp8_block(void* stream, const void* a, const void* a_scales, const void* b, const void* b_scales, int b_block_rows,
                            const void* bias, int bias_is_f32, void* c, int64_t c_stride, int64_t M, int64_t N, int64_t K, float* workspace,
                            int64_t workspace_floats);

#ifdef __cplusplus
}
#endif
#endif /* MDLAYERS_H_ */
