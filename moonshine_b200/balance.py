"""Expert load, balance loss and the router's gradient (``include/k3_moe_balance.h``) on torch tensors.

    router = balance.RouterBalance(experts=896, top_k=16, coefficient=1e-2, route_scale=2.5)
    counts, loss, means = router.forward(logits, ids, offsets)
    d_logits = router.backward(logits, ids, counts, offsets, d_loss, d_weights)
"""
from __future__ import annotations

import torch

from . import ops
from .fp8 import _done, _placed, _Workspace

_SCORES = {"sigmoid": ops.SCORE_SIGMOID, "softmax": ops.SCORE_SOFTMAX}


def _check(t, name, dtype, shape):
    if t.dtype is not dtype or t.shape != shape:
        raise ValueError(f"{name}: expected {dtype} {list(shape)}, got {t.dtype} {list(t.shape)}")


class RouterBalance:
    """``score``: "sigmoid" (the layer's router) or "softmax".  ``offsets`` int32 [sequences + 1] cut the
    tokens into sequences, each with a loss of its own; None: one sequence."""

    def __init__(self, experts: int, top_k: int, score: str = "sigmoid", coefficient: float = 1e-2,
                 route_scale: float = 1.0):
        if score not in _SCORES:
            raise ValueError("score: 'sigmoid' or 'softmax'")
        self.experts, self.top_k, self.score = experts, top_k, _SCORES[score]
        self.coefficient, self.route_scale = float(coefficient), float(route_scale)
        self._workspace = _Workspace(lambda tokens, sequences: ops.k3_moe_balance_workspace_bytes(tokens, sequences, experts))

    def _sequences(self, ids, offsets):
        tokens = ids.shape[0]
        _check(ids, "ids", torch.int32, (tokens, self.top_k))
        if offsets is None:
            return tokens, 1
        if offsets.dtype is not torch.int32 or offsets.dim() != 1 or offsets.shape[0] < 2:
            raise ValueError(f"offsets: expected int32 [sequences + 1], got {offsets.dtype} {list(offsets.shape)}")
        return tokens, offsets.shape[0] - 1

    def forward(self, logits: torch.Tensor | None, ids: torch.Tensor, offsets: torch.Tensor | None = None):
        """logits f32 [tokens, experts], ids int32 [tokens, top_k] -> counts int32 [sequences, experts],
        loss f32 [sequences], means f32 [sequences, experts].  logits None: counts alone."""
        tokens, sequences = self._sequences(ids, offsets)
        if logits is not None:
            _check(logits, "logits", torch.float32, (tokens, self.experts))
        _placed(("ids", ids), ("logits", logits), ("offsets", offsets))
        make = ids.new_empty if tokens else ids.new_zeros
        counts = make((sequences, self.experts))
        loss = means = None
        if logits is not None:
            loss = make(sequences, dtype=torch.float32)
            means = make((sequences, self.experts), dtype=torch.float32)
        if tokens:
            ws = self._workspace.of(tokens, sequences, ids.device)
            _done(ops.k3_moe_balance(counts, loss, means, logits, ids, offsets, tokens, sequences, self.experts, self.top_k,
                                     self.score, self.coefficient, ws, self._workspace.bytes), "k3_moe_balance")
        return counts if logits is None else (counts, loss, means)

    def backward(self, logits: torch.Tensor, ids: torch.Tensor, counts: torch.Tensor | None = None,
                 offsets: torch.Tensor | None = None, d_loss: torch.Tensor | None = None,
                 d_weights: torch.Tensor | None = None) -> torch.Tensor:
        """The gradient by the logits, f32 [tokens, experts], from d_loss f32 [sequences] (with ``counts`` of the
        forward pass) and d_weights f32 [tokens, top_k], of which one may be None."""
        tokens, sequences = self._sequences(ids, offsets)
        _check(logits, "logits", torch.float32, (tokens, self.experts))
        if d_loss is not None:
            _check(d_loss, "d_loss", torch.float32, (sequences,))
            if counts is None:
                raise ValueError("d_loss wants the counts of the forward pass")
            _check(counts, "counts", torch.int32, (sequences, self.experts))
        if d_weights is not None:
            _check(d_weights, "d_weights", torch.float32, (tokens, self.top_k))
        _placed(("ids", ids), ("logits", logits), ("counts", counts), ("offsets", offsets), ("d_loss", d_loss),
                ("d_weights", d_weights))
        d_logits = logits.new_empty((tokens, self.experts))
        if tokens:
            _done(ops.k3_moe_router_backward(d_logits, logits, ids, counts, offsets, d_loss, d_weights, tokens, sequences,
                                             self.experts, self.top_k, self.score, self.coefficient, self.route_scale),
                  "k3_moe_router_backward")
        return d_logits
