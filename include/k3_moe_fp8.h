/*
 * Products on 8-bit floating point tables with one scale per block of 128
 * (CUDA, sm_100a).  No counterpart in the reference: its static weights are
 * Q8-128 and its experts MXFP4; these entry points take checkpoints whose
 * matrices are E4M3 with an f32 scale per 128 x 128 block.  Conventions are
 * those of k3_moe_ops.h: caller-owned device pointers, a cudaStream_t as
 * void *, bool return (false: an invalid argument or a launch error, nothing
 * raised), no allocation, no synchronisation.
 *
 * Formats
 *   codes    E4M3 bytes (largest 448), rows of columns rounded up to 16 bytes
 *            (the pitch); bytes past the columns are written as zeros by the
 *            quantisers and never read as values.  16-byte aligned.
 *   "rows"   f32 scales [rows, p]: one per row and 128 columns, p =
 *            ceil(columns / 128) rounded up to 4.  16-byte aligned.
 *   "blocks" f32 scales [ceil(rows / 128), ceil(columns / 128)], contiguous.
 * A block's scale is max(largest magnitude / 448, 2^-126), a code the quotient
 * value / scale rounded to nearest even, both as f32 divisions.  A block that
 * holds an infinity or a NaN gets the scale NaN and codes NaN, so every
 * result that it enters is NaN.
 *
 * Limits
 *   A product multiplies a block's two scales in f32 before its sum, so that
 *   product keeps its bits between 2^-126 and 2^128 (scales per row on both
 *   sides: the sum times the left one).
 *   Matrices of more than 65535 x 128 rows are refused by the quantisers by
 *   columns and by blocks and by the transposed layout, and as a table by a
 *   product with up to 16 rows.
 */
#ifndef K3_MOE_FP8_H
#define K3_MOE_FP8_H

#include <stdbool.h>
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define K3_MOE_FP8_BF16 0            /* element types of inputs and outputs */
#define K3_MOE_FP8_F32 1
#define K3_MOE_FP8_BLOCKS 0          /* scale layouts of a product's right-hand side */
#define K3_MOE_FP8_ROWS 1

/* x [rows, columns] of x_type -> codes [rows, pitch(columns)] with scales per
 * row.  The left-hand side of a product. */
bool k3_moe_fp8_quantize_rows(void *codes, void *scales, const void *x, uint32_t rows,
                              uint32_t columns, int x_type, void *stream);

/* The same of x transposed: codes [columns, pitch(rows)], scales per column of
 * x and 128 rows.  Both sides of a weight gradient, where the sum runs over
 * tokens. */
bool k3_moe_fp8_quantize_columns(void *codes, void *scales, const void *x, uint32_t rows,
                                 uint32_t columns, int x_type, void *stream);

/* x -> codes [rows, pitch(columns)] with scales per 128 x 128 block: a weight
 * table. */
bool k3_moe_fp8_quantize_blocks(void *codes, void *scales, const void *x, uint32_t rows,
                                uint32_t columns, int x_type, void *stream);

/* A weight table laid out for the gradient by the input: codes [columns,
 * pitch(rows)] and scales [ceil(columns / 128), ceil(rows / 128)] of the
 * transposed matrix, the same values. */
bool k3_moe_fp8_transpose_blocks(void *codes_out, void *scales_out, const void *codes,
                                 const void *scales, uint32_t rows, uint32_t columns,
                                 void *stream);

/* out [m, n] = a [m, k] b [n, k]^T, both as codes; a's scales per row, b's in
 * b_scale_layout.  out is of out_type, contiguous; accumulate != 0 (f32 only)
 * adds to what it holds.  Sums are f32: within a block of 128 on the tensor
 * cores, across blocks scaled and added in ascending order. */
bool k3_moe_fp8_product(void *out, const void *a, const void *a_scales, const void *b,
                        const void *b_scales, uint32_t m, uint32_t n, uint32_t k,
                        int b_scale_layout, int out_type, int accumulate, void *stream);

/* out bf16 [tokens, rows] = x bf16 [tokens, columns] W^T with W [rows, columns]
 * in blocks: quantises x by rows into the workspace and multiplies.  The
 * gradient by the input is this call on dY and the transposed table.  (Here and
 * below the workspace of more tokens serves fewer.) */
size_t k3_moe_fp8_linear_workspace_bytes(uint32_t tokens, uint32_t columns);
bool k3_moe_fp8_linear(void *out, const void *x, const void *w, const void *w_scales,
                       uint32_t tokens, uint32_t rows, uint32_t columns, void *workspace,
                       size_t workspace_bytes, void *stream);

/* dw f32 [rows, columns] = dy bf16 [tokens, rows]^T x bf16 [tokens, columns]
 * (accumulate != 0: added to dw), both quantised by columns within the call. */
size_t k3_moe_fp8_weight_gradient_workspace_bytes(uint32_t tokens, uint32_t rows,
                                                  uint32_t columns);
bool k3_moe_fp8_weight_gradient(void *dw, const void *dy, const void *x, uint32_t tokens,
                                uint32_t rows, uint32_t columns, int accumulate,
                                void *workspace, size_t workspace_bytes, void *stream);

/* Routed experts on such tables. */
typedef struct k3_moe_fp8_experts_desc {
    uint32_t hidden;               /* d, a multiple of 16                          */
    uint32_t expert_hidden;        /* I, a multiple of 16                          */
    uint32_t experts;              /* E <= 1024                                    */
    uint32_t top_k;                /* <= 32                                        */
    int32_t  activation;           /* K3_MOE_ACT_SITU / _SWIGLU (k3_moe_layer.h)   */
    float    beta;                 /* SiTU only                                    */
    float    linear_beta;
    const void *w1;                /* gate [E, I, d] codes                         */
    const void *w1_scales;         /* f32 [E, ceil(I / 128), ceil(d / 128)]        */
    const void *w3;                /* up, as w1                                    */
    const void *w3_scales;
    const void *w2;                /* down [E, d, I] codes                         */
    const void *w2_scales;         /* f32 [E, ceil(d / 128), ceil(I / 128)]        */
} k3_moe_fp8_experts_desc;

/* out bf16 [tokens, d] = sum_r weights[t, r] * expert ids[t, r] of x[t] (bf16
 * [tokens, d]), plus shared bf16 [tokens, d] unless NULL, added as
 * k3_moe_combine does.  ids u32, weights f32 [tokens, top_k] on the device, as
 * k3_moe_route writes them.  Rows are quantised once per token and again after
 * the activation, which is not rounded in between; an expert's output rows are
 * f32 up to their weighted sum, whatever the number of tokens.  An id >= experts
 * contributes nothing and raises bit 1 of k3_moe_device_status(). */
size_t k3_moe_fp8_experts_workspace_bytes(const k3_moe_fp8_experts_desc *desc, uint32_t tokens);
bool k3_moe_fp8_experts_forward(const k3_moe_fp8_experts_desc *desc, void *out, const void *x,
                                const void *ids, const void *weights, const void *shared,
                                uint32_t tokens, void *workspace, size_t workspace_bytes,
                                void *stream);

#ifdef __cplusplus
}
#endif
#endif
