/*
 * Expert load and the training side of the router (CUDA, sm_100a): counts per
 * expert, the balance loss over ragged sequences, and the gradient of that loss
 * and of the routing weights by the router's logits.  No counterpart in the
 * reference, which only serves.  Conventions are those of k3_moe_ops.h.
 *
 * For a token with logits l [E]: scores s = sigmoid(l), total Z = 1e-20 +
 * sum s (K3_MOE_SCORE_SIGMOID, what k3_rocm_router_topk_f32 uses), or s =
 * softmax(l), Z = 1 (K3_MOE_SCORE_SOFTMAX; a row whose logits are all -inf
 * has scores 0).  For a sequence of T tokens with n_e routes to expert e:
 *   f_e = E n_e / (top_k T),  P_e = mean over its tokens of s_e / Z,
 *   loss = coefficient * sum_e f_e P_e        (an empty sequence: 0)
 * and a chosen expert's routing weight is route_scale * s_i / (1e-20 + sum of
 * the token's chosen scores).
 */
#ifndef K3_MOE_BALANCE_H
#define K3_MOE_BALANCE_H

#include <stdbool.h>
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define K3_MOE_SCORE_SIGMOID 0
#define K3_MOE_SCORE_SOFTMAX 1

/* logits f32 [tokens, experts], ids u32 [tokens, top_k], offsets u32
 * [sequences + 1] ascending from 0 to tokens (NULL: one sequence; tokens past
 * the last offset belong to none) -> counts u32 [sequences, experts], loss f32
 * [sequences], means f32 [sequences, experts] (P).  logits, loss and means may
 * be NULL together: counts alone.  An id >= experts is not counted and raises
 * bit 1 of k3_moe_device_status().  experts <= 1024, top_k <= 32,
 * sequences <= 65535.  The workspace of more tokens serves fewer.  Sums run in
 * an order that the numbers of tokens, sequences and experts, the cuts and the
 * logits' alignment decide: the same call gives the same bits.  A score lies
 * within 6e-7 of itself (softmax: besides the f32 rounding of the logit's
 * distance from the row's largest) down to 2^-126, and is 0 below. */
size_t k3_moe_balance_workspace_bytes(uint32_t tokens, uint32_t sequences, uint32_t experts);
bool k3_moe_balance(void *counts, void *loss, void *means, const void *logits, const void *ids,
                    const void *offsets, uint32_t tokens, uint32_t sequences, uint32_t experts,
                    uint32_t top_k, int score, float coefficient, void *workspace,
                    size_t workspace_bytes, void *stream);

/* d_logits f32 [tokens, experts] from d_loss f32 [sequences] (NULL: none) and
 * d_weights f32 [tokens, top_k] (NULL: none; not both).  counts as
 * k3_moe_balance wrote them: the loss's f does not depend on the logits, so
 * nothing else of the forward pass is kept.  An id >= experts has no weight, and
 * raises bit 1 of k3_moe_device_status() where d_weights is given. */
bool k3_moe_router_backward(void *d_logits, const void *logits, const void *ids,
                            const void *counts, const void *offsets, const void *d_loss,
                            const void *d_weights, uint32_t tokens, uint32_t sequences,
                            uint32_t experts, uint32_t top_k, int score, float coefficient,
                            float route_scale, void *stream);

#ifdef __cplusplus
}
#endif
#endif
