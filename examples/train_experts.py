"""A routed block in bf16 that is trained: norm with the residual's addition, router, experts, and all their gradients.

Each step is what a training program runs around one block of a model: the norm (``k3_moe_norm``) hands its rows to the router
in bf16 and to a projection in front of the loss in E4M3, the router (``k3_moe_route``) picks the experts, whose products and
gradients are grouped (``RoutedExperts``); the routing weights' gradient and the balance loss go through ``RouterBalance``
into the router, everything that reached the norm's rows through its backward pass.  The block learns to repeat another
block with other weights.

    python examples/train_experts.py [--steps 40] [--tokens 1024]
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from moonshine_b200 import _native, balance, fp8, grouped, norm, ops      # noqa: E402

HIDDEN, EXPERT_HIDDEN, EXPERTS, TOP_K, BALANCE = 256, 128, 16, 4, 1e-3


class RoutedBlock:
    """out = s + experts(norm(s)), s = x + residual; f32 weights that are trained, bf16 forms that the kernels read."""

    def __init__(self, seed: int):
        g = torch.Generator(device="cuda").manual_seed(seed)
        normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda") * shape[-1] ** -0.5  # noqa: E731
        self.weights = {"w1": normal(EXPERTS, EXPERT_HIDDEN, HIDDEN), "w3": normal(EXPERTS, EXPERT_HIDDEN, HIDDEN),
                        "w2": normal(EXPERTS, HIDDEN, EXPERT_HIDDEN), "norm": torch.ones(HIDDEN, device="cuda"),
                        "router": normal(EXPERTS, HIDDEN)}
        self.read = {name: w.to(torch.bfloat16) for name, w in self.weights.items()}
        self.norm = norm.RmsNorm(self.read["norm"])
        self.experts = grouped.RoutedExperts(self.read["w1"], self.read["w3"], self.read["w2"], TOP_K)
        self.balance = balance.RouterBalance(EXPERTS, TOP_K, coefficient=BALANCE)
        # the router's own products: one group of rows
        self.router, self.by_router = grouped.GroupedProduct(self.read["router"][None]), grouped.GroupedWeightGradient(1, EXPERTS, HIDDEN)
        self.bias = torch.zeros(EXPERTS, device="cuda")
        self.desc = _native.LayerDesc(hidden=HIDDEN, expert_hidden=EXPERT_HIDDEN, expert_count=EXPERTS, top_k=TOP_K,
                                      activation=ops.ACT_SWIGLU, route_scale=1.0, local_expert_first=0, local_expert_count=EXPERTS,
                                      router_weight=self.read["router"].data_ptr(), router_bias=self.bias.data_ptr())

    def forward(self, x: torch.Tensor, residual: torch.Tensor):
        tokens = x.shape[0]
        normed = self.norm.forward(x, residual, y=True, codes=True)
        logits = torch.empty(tokens, EXPERTS, device="cuda")
        ids = torch.empty(tokens, TOP_K, dtype=torch.int32, device="cuda")
        weights = torch.empty(tokens, TOP_K, device="cuda")
        if not ops.k3_moe_route(self.desc, ids, weights, logits, normed.y, tokens):
            raise RuntimeError("k3_moe_route failed")
        routed, saved = self.experts.forward(normed.y, ids, weights)
        return routed, (normed, logits, ids, saved)

    def backward(self, d_routed: torch.Tensor, d_sum: torch.Tensor | None, kept):
        """Gradients by the weights, and by x and the residual."""
        normed, logits, ids, saved = kept
        tokens = ids.shape[0]
        of_experts = self.experts.backward(d_routed, saved)
        counts, loss, _ = self.balance.forward(logits, ids)
        d_logits = self.balance.backward(logits, ids, counts, d_loss=torch.ones_like(loss), d_weights=of_experts.weights).to(torch.bfloat16)
        all_rows = torch.tensor([0, tokens], dtype=torch.int32, device="cuda")
        dy = self.router.by_input(d_logits, all_rows, dtype=torch.float32) + of_experts.x
        dx, d_norm = self.norm.backward(dy.to(torch.bfloat16), normed.sum, normed.rstd, d_sum)
        gradients = {"w1": of_experts.w1, "w3": of_experts.w3, "w2": of_experts.w2, "norm": d_norm,
                     "router": self.by_router.forward(d_logits, normed.y, all_rows)[0]}
        return gradients, dx

    def update(self, gradients: dict, rate: float):
        for name, g in gradients.items():
            self.weights[name] -= rate * g
            self.read[name].copy_(self.weights[name])


def main(steps: int = 40, tokens: int = 1024, rate: float = 2.0, seed: int = 1, quiet: bool = False):
    block, taught = RoutedBlock(seed), RoutedBlock(seed + 100)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    # a projection that reads the norm's E4M3 rows: what a next layer in 8 bits would take
    table, scales = fp8.quantize_blocks(torch.randn(HIDDEN, HIDDEN, generator=g, device="cuda") * HIDDEN ** -0.5)
    projection = fp8.Fp8Linear(table, scales, HIDDEN, HIDDEN)
    losses = []
    for i in range(steps):
        x, residual = (torch.randn(tokens, HIDDEN, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
        want, _ = taught.forward(x, residual)
        got, kept = block.forward(x, residual)
        error = got.float() - want.float()
        losses.append(float(error.square().mean()))
        gradients, dx = block.backward((2 / tokens * error).to(torch.bfloat16), None, kept)
        if not torch.isfinite(projection.forward_codes(kept[0].codes, kept[0].scales)).all() or not torch.isfinite(dx).all():
            raise RuntimeError("a result is not finite")
        block.update(gradients, rate / HIDDEN)
        if not quiet and (i % 10 == 0 or i + 1 == steps):
            print(f"step {i:3d}: mean squared error {losses[-1]:.5f}")
    return losses


if __name__ == "__main__":
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--steps", type=int, default=40)
    p.add_argument("--tokens", type=int, default=1024)
    a = p.parse_args()
    main(a.steps, a.tokens)
