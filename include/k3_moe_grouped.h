/*
 * bf16 products grouped by expert with ragged sizes, and their gradients
 * (CUDA, sm_100a): what routed experts in bf16 are trained and served with.  No
 * counterpart in the reference, whose experts are MXFP4 and frozen.  Conventions
 * are those of k3_moe_ops.h: caller-owned device pointers, a cudaStream_t as
 * void *, bool return (false: an invalid argument or a launch error, nothing
 * raised), no allocation, no synchronisation.
 *
 * Rows are sorted by group, as k3_moe_dispatch_build and k3_rocm_gather_rows_bf16
 * leave them: group g has the rows offsets[g] .. offsets[g + 1] - 1, offsets u32
 * [groups + 1] ascending on the device.  Group sizes are not known to the host
 * and may be anything, zero too.  Rows in front of offsets[0] and from
 * offsets[groups] on belong to no group: they are not written, and what they
 * hold (NaN, say) enters nothing.  An offset past `rows` counts as `rows`, one
 * below its predecessor ends an empty group; nothing outside is read or written.
 * (Where offsets descend, groups may overlap: a row of several has the result of
 * any of them, and rows may be left as they are.)
 *
 * Sums are f32, rounded once to the output's type.  The tensor cores cut an
 * addition of 16 products off instead of rounding it; f32 outputs of theirs lie
 * about 5e-7 of their norm from the exact ones whatever the depth, those of the
 * FMA pipes about 2e-7.  A bf16 output is the rounding of a sum that lies up to
 * 1.2e-9 of the norm off per step of the depth (8e-6 at 7168), so one in some
 * hundreds is the neighbour of the nearest.
 * The order of the sums depends on the sizes of the call and the size of the
 * row's group, not on which SM takes what: the same call gives the same bits.
 * What is not finite in a row or a matrix makes the results that it enters not
 * finite, and no others.
 *
 * Any n and k are taken.  Matrices whose rows are whole units of 16 bytes (n and
 * k multiples of 8, 16-byte aligned pointers) run on the tensor cores, others on
 * the FMA pipes at a fraction of the speed.
 *
 * out_type bf16 or f32; accumulate != 0 (f32 only) adds to what the output
 * holds.  groups <= 1024.  The workspace (16-byte aligned) needs no
 * initialisation; calls that share one have to be ordered.
 */
#ifndef K3_MOE_GROUPED_H
#define K3_MOE_GROUPED_H

#include <stdbool.h>
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define K3_MOE_GROUPED_BF16 0        /* element types of outputs */
#define K3_MOE_GROUPED_F32 1

/* The workspace of any call below, 0 for sizes that are refused.  The workspace
 * of more rows or groups serves fewer. */
size_t k3_moe_grouped_workspace_bytes(uint32_t rows, uint32_t groups);

/* out [rows, n]: out[r] = W_g x[r] for r in group g; x bf16 [rows, k], w bf16
 * [groups, n, k]. */
bool k3_moe_grouped_product(void *out, const void *x, const void *w, const void *offsets,
                            uint32_t rows, uint32_t groups, uint32_t n, uint32_t k, int out_type,
                            int accumulate, void *workspace, size_t workspace_bytes, void *stream);

/* Its gradient by the input, from the same matrices: dx [rows, k]: dx[r] =
 * W_g^T dy[r]; dy bf16 [rows, n]. */
bool k3_moe_grouped_by_input(void *dx, const void *dy, const void *w, const void *offsets,
                             uint32_t rows, uint32_t groups, uint32_t n, uint32_t k, int out_type,
                             int accumulate, void *workspace, size_t workspace_bytes, void *stream);

/* Its gradient by the matrices: dw [groups, n, k]: dw_g = sum over the group's
 * rows of dy[r] x[r]^T, zeros for a group without rows (accumulate != 0: left as
 * they are). */
bool k3_moe_grouped_by_weight(void *dw, const void *dy, const void *x, const void *offsets,
                              uint32_t rows, uint32_t groups, uint32_t n, uint32_t k, int out_type,
                              int accumulate, void *workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif
