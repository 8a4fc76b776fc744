/*
 * RMS norm with the residual's addition in front and E4M3 codes behind, and its
 * gradient (CUDA, sm_100a).  k3_rocm_rms_norm_bf16 (k3_moe_ops.h) normalises
 * bf16 rows to bf16; these entry points also take the addition, f32 rows, and
 * write what an 8-bit product reads (k3_moe_fp8.h) in the same pass.
 * Conventions are those of k3_moe_ops.h.
 *
 *   s    = x + residual, rounded to the element type
 *   rstd = 1 / sqrt(mean of s^2 over the row + epsilon)
 *   y    = s rstd weight
 * y is f32 until it is stored: bf16 rows are y rounded once, codes are those of
 * y itself with a scale per row and 128 columns (format "rows" of
 * k3_moe_fp8.h).  Of bf16 x they are the exact ones: the rounding of 448 s weight /
 * max |s weight| of the block, ties to even.  A block of 128 that is not finite
 * gets the scale NaN.  Where the sum of a row's squares passes f32's range, from
 * |s| of about 1e17 on, rstd is 0.
 * Sums are f32; their order depends on hidden and, where it is no multiple of 8,
 * on the row's place modulo 8: the same call gives the same bits.
 */
#ifndef K3_MOE_NORM_H
#define K3_MOE_NORM_H

#include <stdbool.h>
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define K3_MOE_NORM_BF16 0           /* element types of x, residual, sum and their gradients */
#define K3_MOE_NORM_F32 1

/* x, residual (NULL: none) and sum (NULL: not wanted; may be x or residual
 * itself) [rows, hidden] of `type`, weight bf16 [hidden]; y bf16 [rows, hidden]
 * or NULL; codes [rows, hidden rounded up to 16], 16-byte aligned, with scales
 * f32 [rows, ceil(hidden / 128) rounded up to 4], or both NULL; rstd f32 [rows]
 * or NULL.  One of y and codes at least.  hidden <= 16384, epsilon > 0. */
bool k3_moe_norm(void *sum, void *y, void *codes, void *scales, void *rstd, const void *x,
                 const void *residual, const void *weight, uint32_t rows, uint32_t hidden, int type,
                 float epsilon, void *stream);

/* dx [rows, hidden] of `type`, the gradient by x and by the residual alike, from
 * dy bf16 [rows, hidden], the forward pass's sum (or x) and rstd, and d_sum
 * [rows, hidden] of `type`, what the sum's other readers send back (NULL: none;
 * may be dx itself); d_weight f32 [hidden] or NULL:
 *   dx = d_sum + rstd (weight dy - s rstd^2 mean(weight dy s))
 *   d_weight = sum over rows of dy s rstd, or added to d_weight (accumulate != 0)
 * Sums are f32 in an order that the sizes decide.  The workspace (16-byte
 * aligned) is for d_weight; that of more rows serves fewer.  rows 0: d_weight is
 * zeros, or left as it is. */
size_t k3_moe_norm_workspace_bytes(uint32_t rows, uint32_t hidden);
bool k3_moe_norm_backward(void *dx, void *d_weight, const void *dy, const void *sum, const void *rstd,
                          const void *d_sum, const void *weight, uint32_t rows, uint32_t hidden,
                          int type, int accumulate, void *workspace, size_t workspace_bytes,
                          void *stream);

#ifdef __cplusplus
}
#endif
#endif
