"""A routed layer on E4M3 experts whose router is trained until its load is even.

Each step is what a training program runs around frozen experts in 8 bits: the router (``k3_moe_route``),
the routed experts on E4M3 tables, counts per expert and balance loss, the gradient by the router's
logits, the router weight's gradient by an E4M3 product over the tokens, and an update of the weight.
A projection in the same format stands in front, as the latent projection of the layer does.

    python examples/balance_router_fp8.py [--steps 60] [--tokens 2048]
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from moonshine_b200 import _native, balance, fp8, ops      # noqa: E402

MODEL, HIDDEN, EXPERT_HIDDEN, EXPERTS, TOP_K = 1024, 512, 256, 64, 8


def expert_tables(g: torch.Generator):
    """Tables of all experts and their scales, quantised expert by expert."""
    tables = []
    for rows, columns in ((EXPERT_HIDDEN, HIDDEN), (EXPERT_HIDDEN, HIDDEN), (HIDDEN, EXPERT_HIDDEN)):
        parts = [fp8.quantize_blocks(torch.randn(rows, columns, generator=g, device="cuda", dtype=torch.bfloat16) * columns ** -0.5)
                 for _ in range(EXPERTS)]
        tables += [torch.stack([p[0] for p in parts]), torch.stack([p[1] for p in parts])]
    return tables


class RoutedLayer:
    def __init__(self, seed: int):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.experts = fp8.Fp8Experts(*expert_tables(g), top_k=TOP_K, activation="swiglu")
        projection = torch.randn(HIDDEN, MODEL, generator=g, device="cuda", dtype=torch.bfloat16) * MODEL ** -0.5
        self.project = fp8.Fp8Linear(*fp8.quantize_blocks(projection), HIDDEN, MODEL)
        # the router: an f32 weight that is trained, its bf16 form that the layer reads; some experts start far ahead
        self.weight = torch.randn(EXPERTS, HIDDEN, generator=g, device="cuda") * 0.02
        self.weight[:EXPERTS // 8] += torch.randn(HIDDEN, generator=g, device="cuda") * 0.05
        self.router_weight = self.weight.to(torch.bfloat16)
        self.bias = torch.zeros(EXPERTS, device="cuda")
        self.desc = _native.LayerDesc(
            hidden=HIDDEN, expert_hidden=EXPERT_HIDDEN, expert_count=EXPERTS, top_k=TOP_K, activation=ops.ACT_SWIGLU,
            route_scale=1.0, local_expert_first=0, local_expert_count=EXPERTS, router_weight=self.router_weight.data_ptr(),
            router_bias=self.bias.data_ptr())
        self.balance = balance.RouterBalance(EXPERTS, TOP_K, coefficient=1.0)
        # by_weight() alone is used: the transposed table of the router is not needed for it
        codes, scales = fp8.quantize_blocks(self.router_weight)
        self.router_gradient = fp8.Fp8LinearGradient(*fp8.transpose_blocks(codes, scales, EXPERTS, HIDDEN), EXPERTS, HIDDEN)

    def forward(self, x: torch.Tensor):
        """x bf16 [tokens, MODEL] -> (latent, logits, ids, out)."""
        latent = self.project.forward(x)
        tokens = x.shape[0]
        logits = torch.empty(tokens, EXPERTS, device="cuda")
        ids = torch.empty(tokens, TOP_K, dtype=torch.int32, device="cuda")
        weights = torch.empty(tokens, TOP_K, device="cuda")
        if not ops.k3_moe_route(self.desc, ids, weights, logits, latent, tokens):
            raise RuntimeError("k3_moe_route failed")
        return latent, logits, ids, self.experts.forward(latent, ids, weights)

    def step(self, x: torch.Tensor, offsets: torch.Tensor, rate: float):
        """One pass and one update of the router; the mean loss of the sequences and the counts of all tokens."""
        latent, logits, ids, out = self.forward(x)
        counts, loss, _ = self.balance.forward(logits, ids, offsets)
        d_loss = torch.full_like(loss, 1.0 / loss.numel())
        d_logits = self.balance.backward(logits, ids, counts, offsets, d_loss=d_loss)
        gradient = self.router_gradient.by_weight(d_logits.to(torch.bfloat16), latent)
        self.weight -= rate * gradient
        self.router_weight.copy_(self.weight)
        return float(loss.mean()), counts.sum(0), out


def main(steps: int = 60, tokens: int = 2048, rate: float = 4.0, seed: int = 1, quiet: bool = False):
    layer = RoutedLayer(seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    cuts = torch.tensor([0, tokens // 5, tokens // 2, tokens - tokens // 7, tokens], dtype=torch.int32, device="cuda")
    loads = []
    for i in range(steps):
        x = torch.randn(tokens, MODEL, generator=g, device="cuda", dtype=torch.bfloat16) + 0.5
        loss, counts, out = layer.step(x, cuts, rate)
        loads.append(float(counts.max()) / float(counts.float().mean()))
        if not torch.isfinite(out).all():
            raise RuntimeError("the layer's output is not finite")
        if not quiet and (i % 10 == 0 or i + 1 == steps):
            print(f"step {i:3d}: balance loss {loss:.4f}, most loaded expert {loads[-1]:.2f} times the mean")
    return loads


if __name__ == "__main__":
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--steps", type=int, default=60)
    p.add_argument("--tokens", type=int, default=2048)
    a = p.parse_args()
    main(a.steps, a.tokens)
