/*
 * hcg_lm.h -- C ABI of the language-model operators of the gfx950 backend:
 * the embedding lookup, layer norm, root-mean-square norm and the softmax cross
 * entropy of a linear head, each with its gradient.  They stand next to the products of
 * hcg_gemm.h (same library, status codes, error text and stream rules) and
 * have no counterpart in the reference, whose only data-parallel path is the
 * tiled product.
 *
 * Matrices are row-major, with the row stride in elements; nothing but scratch
 * needs an alignment beyond its elements'.  Element types are HCG_F16, HCG_BF16
 * (hcg_gemm.h) or HCG_F32.  Sums and statistics are float32; a 16-bit output
 * is rounded once (to nearest, ties to even); hcg_linear_cross_entropy_grad
 * holds two intermediates in 16 bits, see there.  Every result is
 * bit-reproducible.
 *
 * Scratch is the caller's: a call that needs some has a ..._workspace
 * function for its size in bytes, takes 256-byte aligned device memory of at
 * least that size and leaves nothing in it.  No entry point allocates, copies
 * to the host or waits, so all of them can be captured into a HIP graph.
 */
#ifndef HCG_LM_H
#define HCG_LM_H

#include <stdint.h>

#include "hcg_gemm.h"

#ifdef __cplusplus
extern "C" {
#endif

#define HCG_F32 2 /* beside HCG_F16 and HCG_BF16 of hcg_gemm.h */

/* out[i] = scale * table[ids[i]] for i < n, one float32 product per element.
 * ids are 32- or 64-bit (id_bytes 4 or 8); an id outside [0, vocab) gives a
 * row of NaN (nothing outside the table is read).  Bound: HBM. */
int hcg_embedding(int dtype, const void* table, int64_t ldt, int64_t vocab, int64_t width, int id_bytes,
                  const void* ids, int64_t n, float scale, void* out, int64_t ldo, void* stream);

/* grad[v] = scale * sum of dy[i] over the i with ids[i] == v, for every v <
 * vocab (rows without an i, and row padding_idx, are zeros; padding_idx < 0:
 * none; an id outside [0, vocab) reaches no row).  dy is n x width of dtype,
 * grad vocab x width of grad_dtype (dtype or HCG_F32).  The sum of a row is
 * float32 over ascending i, in fixed pieces where it is long.  n and vocab are
 * below 2^28, width below 2^23. */
int64_t hcg_embedding_grad_workspace(int dtype, int64_t n, int64_t vocab, int64_t width);
int hcg_embedding_grad(int dtype, const void* dy, int64_t ldy, int64_t n, int64_t width, int id_bytes,
                       const void* ids, int64_t vocab, int64_t padding_idx, float scale, int grad_dtype,
                       void* grad, int64_t ldg, void* workspace, int64_t workspace_bytes, void* stream);

/* y = (x - mean) * rstd * weight + bias by rows, rstd = 1 / sqrt(var + eps)
 * with the biased variance (two passes over registers).  weight and bias
 * (param_dtype, width elements) may be null; mean and rstd (float32, one per
 * row) may be null. */
int hcg_layer_norm(int dtype, const void* x, int64_t ldx, int64_t rows, int64_t width, int param_dtype,
                   const void* weight, const void* bias, float eps, void* y, int64_t ldy, float* mean, float* rstd,
                   void* stream);

/* The gradients of hcg_layer_norm: dx (dtype), dweight = sum over rows of
 * dy * xhat and dbias = sum of dy (param_dtype; either may be null). */
int64_t hcg_layer_norm_grad_workspace(int64_t rows, int64_t width);
int hcg_layer_norm_grad(int dtype, const void* dy, int64_t lddy, const void* x, int64_t ldx, int64_t rows,
                        int64_t width, const float* mean, const float* rstd, int param_dtype, const void* weight,
                        void* dx, int64_t lddx, void* dweight, void* dbias, void* workspace, int64_t workspace_bytes,
                        void* stream);

/* y = h * rstd * weight by rows, rstd = 1 / sqrt(mean of h^2 + eps).  h = x +
 * residual, rounded to residual_dtype (dtype or HCG_F32) and written to h, which
 * may be the residual itself; without one (null) h is x and is not written.
 * weight (param_dtype: dtype or HCG_F32, width elements) and rstd (float32, one
 * per row) may be null. */
int hcg_rms_norm(int dtype, const void* x, int64_t ldx, int64_t rows, int64_t width, int residual_dtype,
                 const void* residual, int64_t ldr, int param_dtype, const void* weight, float eps, void* y,
                 int64_t ldy, void* h, int64_t ldh, float* rstd, void* stream);

/* The gradients of hcg_rms_norm for x and the residual, which are one: dh =
 * rstd * (dy * weight - h * rstd * mean of (dy * weight * h * rstd)) + dresidual
 * (h_dtype: dtype or HCG_F32, as h and dresidual, the gradient that reaches h
 * past the norm; may be null), and dweight = sum over rows of dy * h * rstd
 * (param_dtype; may be null, and so may weight).  dh may be dresidual itself. */
int64_t hcg_rms_norm_grad_workspace(int64_t rows, int64_t width);
int hcg_rms_norm_grad(int dtype, const void* dy, int64_t lddy, int h_dtype, const void* h, int64_t ldh, int64_t rows,
                      int64_t width, const float* rstd, int param_dtype, const void* weight, const void* dresidual,
                      int64_t lddr, void* dh, int64_t lddh, void* dweight, void* workspace, int64_t workspace_bytes,
                      void* stream);

/* Softmax cross entropy of the logits x @ weight^T against one target per
 * row, without the logits in memory.  x: tokens x width, weight: vocab x
 * width (dtype HCG_F16 or HCG_BF16), targets 32- or 64-bit.  Per row,
 * lse = log sum_v exp(x . weight[v]) and loss = lse - x . weight[target];
 * both 0 where target == ignore_index (such a row may hold anything, NaN too).
 * A target outside [0, vocab) that is not ignore_index gives a NaN loss (and
 * no one-hot term in a gradient).  The workspace's size depends on the
 * weight's alignment: rows that are not 16-byte aligned are copied there.
 * tokens are below 2^26, vocab and width below 4,000,000 - 8. */
int64_t hcg_linear_cross_entropy_workspace(int64_t tokens, int64_t vocab, int64_t width, const void* weight,
                                           int64_t ldw, int grad);
int hcg_linear_cross_entropy(int dtype, const void* x, int64_t ldx, int64_t tokens, const void* weight, int64_t ldw,
                             int64_t vocab, int64_t width, int id_bytes, const void* targets, int64_t ignore_index,
                             float* loss, float* lse, void* workspace, int64_t workspace_bytes, void* stream);

/* The sum of the losses (mean = 0) or their mean over the rows that count
 * (mean = 1; 0 when none does) into *loss, and the gradients of grad_scale
 * times it: dx (tokens x width) and dweight (vocab x width), of dtype.  Between
 * the products, exponentials are held as f16 (within 2^-11 of the value, or
 * 2^-40 of the largest among the 32 to 128 words they are computed with; 2^-25
 * where logits pass 7e5) and
 * probabilities minus the one-hot in dtype (HCG_F16: times 2^15, so 2^-40 near
 * zero): beside the result's own rounding, as much again where few tokens or
 * words enter a sum.  They take scratch of 2 bytes per word for up to 2^29 words
 * (1 GiB, and the rows' padding), or 256 tokens if those have more. */
int hcg_linear_cross_entropy_grad(int dtype, const void* x, int64_t ldx, int64_t tokens, const void* weight,
                                  int64_t ldw, int64_t vocab, int64_t width, int id_bytes, const void* targets,
                                  int64_t ignore_index, int mean, float grad_scale, float* loss, void* dx,
                                  int64_t lddx, void* dweight, int64_t lddw, void* workspace,
                                  int64_t workspace_bytes, void* stream);

/* How calls of these sizes run (no device is asked): plan[0] is the number of
 * pieces that the tokens are taken in; then, for the logits (vocab x tokens)
 * and, where grad is not 0, dx (width x tokens) and dweight (width x vocab),
 * three values each: a tile's rows, its columns, and the parts that the sums
 * are split into if every token of a piece counts.  plan has room for 10. */
int hcg_linear_cross_entropy_plan(int64_t tokens, int64_t vocab, int64_t width, int grad, int* plan);

#ifdef __cplusplus
}
#endif

#endif /* HCG_LM_H */
