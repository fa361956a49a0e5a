/*
 * hcg_fp8.h -- C ABI of the 8-bit linear layers of the gfx950 backend: the
 * product of two matrices in 8-bit floating point, the quantiser that makes
 * them, and the root-mean-square norm that writes its result quantised.  They
 * stand next to the operators of hcg_lm.h (same library, status codes, error
 * text, stream and scratch rules) and have no counterpart in the reference.
 *
 * A quantised matrix is rows x cols elements of HCG_E4M3 (1 sign, 4 exponent, 3
 * mantissa bits; largest value 448, no infinities) or HCG_E5M2 (largest 57344),
 * row-major with the row stride in bytes, and a scale for each 128 columns (the
 * last block may be shorter) of each row, or of each 128 rows (tiles).  Element
 * (r, c) stands for q[r][c] * scale[r or r / 128][c / 128].  Scales are HCG_F32,
 * or HCG_E8M0: the power of two 2^(byte - 127), 255 a NaN.  They lie where two
 * strides (in elements) put them: scale[i * scale_row + j * scale_block].
 *
 * Quantising: a = max(largest |x| of the block, 2^-100); an HCG_F32 scale is
 * a / F, F the type's largest value, and q = x * (F / a) rounded to nearest,
 * ties to even (each quotient one float32 rounding); an HCG_E8M0 scale is the
 * least power of two that is not below a / F, and q = x / scale rounded.  A block
 * that holds an infinity or a NaN stands for NaN, all of it.
 */
#ifndef HCG_FP8_H
#define HCG_FP8_H

#include <stdint.h>

#include "hcg_lm.h"

#ifdef __cplusplus
extern "C" {
#endif

#define HCG_E4M3 3 /* beside HCG_F16, HCG_BF16 and HCG_F32 */
#define HCG_E5M2 4
#define HCG_E8M0 5 /* scales only */

#define HCG_FP8_BLOCK 128 /* columns (and rows of a tile) that share a scale */

/* q and scale of x (rows x cols, of dtype HCG_F16, HCG_BF16 or HCG_F32), or with
 * transpose of its transpose (q is then cols x rows).  tile: one scale per 128 x
 * 128 tile, else per row and 128 columns, of the matrix that q is.  Bound: HBM.
 * rows and cols are below 2^31. */
int hcg_quantize_fp8(int dtype, const void* x, int64_t ldx, int64_t rows, int64_t cols, int transpose, int tile,
                     int q_dtype, void* q, int64_t ldq, int scale_dtype, void* scale, int64_t scale_row,
                     int64_t scale_block, void* stream);

/* hcg_rms_norm (hcg_lm.h) with the result quantised by rows before any other
 * rounding: q and scale stand for h * rstd * weight. */
int hcg_rms_norm_fp8(int dtype, const void* x, int64_t ldx, int64_t rows, int64_t width, int residual_dtype,
                     const void* residual, int64_t ldr, int param_dtype, const void* weight, float eps, int q_dtype,
                     void* q, int64_t ldq, int scale_dtype, void* scale, int64_t scale_row, int64_t scale_block,
                     void* h, int64_t ldh, float* rstd, void* stream);

/* y = x @ weight^T: x is tokens x inputs (HCG_E4M3 or HCG_E5M2) scaled by rows,
 * weight outputs x inputs (HCG_E4M3) scaled by tiles (w_tile) or by rows, y
 * tokens x outputs of out_dtype (HCG_F16, HCG_BF16 or HCG_F32).  The products of
 * each 128 inputs are added up in float32, times both scales (their float32
 * product), and so are the blocks.  For a HCG_F32 y the products are exact.  A
 * 16-bit y is rounded once, and its products come from the 8-bit matrix
 * instructions, which cut each of 8 neighbours below 2^-13 of the largest of them:
 * 1.5e-5 of the results for normal operands, up to 8e-5 where a few columns are much
 * larger than the others, at most 2^-10 of the sum of magnitudes.  (With HCG_E8M0
 * scales these instructions multiply by them and add up all of inputs.)  Operands
 * need no alignment; rows that start at multiples of 16 bytes are read where they lie,
 * others may be copied to scratch first.  inputs and the row strides are below
 * 4,000,000, tokens and outputs below 2^26.
 *
 * algo: HCG_FP8_AUTO picks by the sizes; the others are for tests and
 * measurements. */
#define HCG_FP8_AUTO 0
#define HCG_FP8_STREAM 1 /* operands straight into registers, any alignment */
#define HCG_FP8_256x256 2 /* tiles of outputs x tokens; 128x128 for float32 results and weights scaled by rows in float32 */
#define HCG_FP8_128x128 3
#define HCG_FP8_128x64 4
#define HCG_FP8_SPLITS 256 /* times a number up to 16, added to a form: K in so many parts */

/* (0 for sizes and forms that hcg_linear_fp8 refuses, which says why.) */
int64_t hcg_linear_fp8_workspace(int algo, int64_t tokens, int64_t outputs, int64_t inputs, const void* x, int64_t ldx,
                                 const void* weight, int64_t ldw, int scale_dtype, int64_t xs_row, int w_tile,
                                 const void* w_scale, int64_t ws_row, int64_t ws_block, int out_dtype);
int hcg_linear_fp8(int algo, int x_dtype, const void* x, int64_t ldx, int64_t tokens, const void* weight, int64_t ldw,
                   int64_t outputs, int64_t inputs, int scale_dtype, const void* x_scale, int64_t xs_row,
                   int64_t xs_block, int w_tile, const void* w_scale, int64_t ws_row, int64_t ws_block, int out_dtype,
                   void* y, int64_t ldy, void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* HCG_FP8_H */
