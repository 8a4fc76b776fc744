"""Routed experts in bf16 that can be trained: products grouped by expert with their gradients
(``include/k3_moe_grouped.h``) and the gated activation with its gradient, on torch tensors.

Rows are sorted by expert, as ``k3_moe_dispatch_build`` and ``k3_rocm_gather_rows_bf16`` leave them;
``offsets`` int32 [groups + 1] on the device say where each group's rows begin.  Rows outside
``offsets[0] .. offsets[groups]`` are not written: a new tensor holds anything there, and an ``out`` given
to a call keeps what it has.  An object keeps a workspace as those of ``fp8`` do; all tensors of a call lie
on the current CUDA device.

    up = grouped.GroupedProduct(w1)                         # bf16 [experts, n, k]
    y = up.forward(x, offsets)                              # [rows, k] -> [rows, n]
    dx = up.by_input(dy, offsets, dtype=torch.float32)
    dw = grouped.GroupedWeightGradient(experts, n, k).forward(dy, x, offsets)
    d_gate, d_up, scaled, d_weights = grouped.GatedActivation("swiglu").backward(d_out, gate, up, weights, routes)
"""
from __future__ import annotations

import torch

from . import ops
from .balance import _check
from .fp8 import _ACTIVATIONS, _done, _matrix, _placed, _Workspace

_OUT = {torch.bfloat16: ops.GROUPED_BF16, torch.float32: ops.GROUPED_F32}


def _output(like, shape, dtype, out, into):
    """The tensor that a call writes (out), adds to (into) or makes, and whether it adds."""
    if out is not None and into is not None:
        raise ValueError("out and into: one of them")
    if into is not None:
        _check(into, "into", torch.float32, shape)
        return into, 1
    if out is not None:
        if out.dtype not in _OUT or out.shape != shape:
            raise ValueError(f"out: expected bfloat16 or float32 {list(shape)}, got {out.dtype} {list(out.shape)}")
        return out, 0
    if dtype not in _OUT:
        raise ValueError(f"dtype: bfloat16 or float32, got {dtype}")
    return None, 0


class GroupedProduct:
    """y = x W_g^T for the rows of each group g, and dx = dy W_g, for bf16 matrices ``w`` [groups, n, k]."""

    def __init__(self, w: torch.Tensor):
        if w.dim() != 3 or w.dtype is not torch.bfloat16 or not w.is_contiguous():
            raise ValueError(f"w: expected contiguous bfloat16 [groups, n, k], got {w.dtype} {list(w.shape)}")
        self.w, self._device = w, w.device
        self.groups, self.n, self.k = w.shape
        self._workspace = _Workspace(lambda rows: ops.k3_moe_grouped_workspace_bytes(rows, self.groups))

    def _run(self, name, call, x, wide, columns, offsets, dtype, out, into):
        rows, _ = _matrix(x, name, wide)
        _check(offsets, "offsets", torch.int32, (self.groups + 1,))
        to, add = _output(x, (rows, columns), dtype, out, into)
        _placed((name, x), ("offsets", offsets), ("out", out), ("into", into), tables=self._device)
        if to is None:
            to = x.new_empty((rows, columns), dtype=dtype)
        if rows:
            ws = self._workspace.of(rows, x.device)
            _done(getattr(ops, call)(to, x, self.w, offsets, rows, self.groups, self.n, self.k, _OUT[to.dtype], add, ws,
                                     self._workspace.bytes), call)
        return to

    def forward(self, x: torch.Tensor, offsets: torch.Tensor, dtype: torch.dtype = torch.bfloat16,
                out: torch.Tensor | None = None, into: torch.Tensor | None = None) -> torch.Tensor:
        """x bf16 [rows, k] -> [rows, n] of ``dtype`` (bf16 or f32), written to ``out``, or added to ``into`` (f32)."""
        return self._run("x", "k3_moe_grouped_product", x, self.k, self.n, offsets, dtype, out, into)

    def by_input(self, dy: torch.Tensor, offsets: torch.Tensor, dtype: torch.dtype = torch.bfloat16,
                 out: torch.Tensor | None = None, into: torch.Tensor | None = None) -> torch.Tensor:
        """dy bf16 [rows, n] -> dx [rows, k], as ``forward``."""
        return self._run("dy", "k3_moe_grouped_by_input", dy, self.n, self.k, offsets, dtype, out, into)


class GroupedWeightGradient:
    """dW_g = sum of dy[r]^T x[r] over the rows of each group."""

    def __init__(self, groups: int, n: int, k: int):
        self.groups, self.n, self.k = groups, n, k
        self._workspace = _Workspace(lambda rows: ops.k3_moe_grouped_workspace_bytes(rows, groups))

    def forward(self, dy: torch.Tensor, x: torch.Tensor, offsets: torch.Tensor, dtype: torch.dtype = torch.float32,
                out: torch.Tensor | None = None, into: torch.Tensor | None = None) -> torch.Tensor:
        """dy bf16 [rows, n], x bf16 [rows, k] -> [groups, n, k] of ``dtype``, written to ``out``, or added to ``into``
        (f32).  A group without rows gets zeros (``into``: stays)."""
        rows, _ = _matrix(dy, "dy", self.n)
        if _matrix(x, "x", self.k)[0] != rows:
            raise ValueError("dy and x: different numbers of rows")
        _check(offsets, "offsets", torch.int32, (self.groups + 1,))
        shape = (self.groups, self.n, self.k)
        to, add = _output(dy, shape, dtype, out, into)
        _placed(("dy", dy), ("x", x), ("offsets", offsets), ("out", out), ("into", into))
        if rows == 0:
            if to is None:
                return dy.new_zeros(shape, dtype=dtype)
            return to if add else to.zero_()
        if to is None:
            to = dy.new_empty(shape, dtype=dtype)
        ws = self._workspace.of(rows, dy.device)
        _done(ops.k3_moe_grouped_by_weight(to, dy, x, offsets, rows, self.groups, self.n, self.k, _OUT[to.dtype], add, ws,
                                           self._workspace.bytes), "k3_moe_grouped_by_weight")
        return to


class GatedActivation:
    """act = activation(gate) up ("swiglu", or "situ" with its bounds) between an expert's products."""

    def __init__(self, activation: str = "swiglu", beta: float = 4.0, linear_beta: float = 25.0):
        if activation not in _ACTIVATIONS:
            raise ValueError("activation: 'swiglu' or 'situ'")
        self.activation, self.beta, self.linear_beta = _ACTIVATIONS[activation], float(beta), float(linear_beta)

    def forward(self, gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
        """gate, up bf16 [rows, columns] -> bf16 [rows, columns]."""
        rows, columns = _matrix(gate, "gate")
        _check(up, "up", torch.bfloat16, (rows, columns))
        _placed(("gate", gate), ("up", up))
        out = torch.empty_like(gate)
        if rows and columns:
            _done(ops.k3_moe_activation_bf16(out, gate, up, rows * columns, self.activation, self.beta, self.linear_beta),
                  "k3_moe_activation_bf16")
        return out

    def backward(self, d_out: torch.Tensor, gate: torch.Tensor, up: torch.Tensor, weights: torch.Tensor | None = None,
                 routes: torch.Tensor | None = None, offsets: torch.Tensor | None = None):
        """d_out, gate, up bf16 [rows, columns] -> d_gate, d_up, scaled (bf16) and d_weights.

        Row r belongs to route ``routes[r]`` (int32 [rows], each route once; None: route r), whose routing weight is
        that element of ``weights`` (f32, [tokens, top_k] say; None: 1 for each row).  ``d_out`` is the gradient that the
        down matrix sends back for the unweighted row; ``scaled``, weight times activation, is what that matrix's own
        gradient reads.  d_weights f32 has the shape of ``weights``, [rows] without them.  With ``offsets`` rows outside of
        the groups are left out."""
        rows, columns = _matrix(d_out, "d_out")
        _check(gate, "gate", torch.bfloat16, (rows, columns))
        _check(up, "up", torch.bfloat16, (rows, columns))
        if weights is not None and (weights.dtype is not torch.float32 or (routes is None and weights.numel() != rows)):
            raise ValueError(f"weights: expected float32, one for each of {rows} rows or with routes, got {weights.dtype} "
                             f"{list(weights.shape)}")
        if routes is not None:
            _check(routes, "routes", torch.int32, (rows,))
        if offsets is not None and (offsets.dtype is not torch.int32 or offsets.dim() != 1 or offsets.shape[0] < 2):
            raise ValueError(f"offsets: expected int32 [groups + 1], got {offsets.dtype} {list(offsets.shape)}")
        _placed(("d_out", d_out), ("gate", gate), ("up", up), ("weights", weights), ("routes", routes), ("offsets", offsets))
        d_gate, d_up, scaled = torch.empty_like(d_out), torch.empty_like(d_out), torch.empty_like(d_out)
        count = rows if weights is None else weights.numel()
        # routes that no row has get no gradient
        if offsets is None and count == rows and rows and columns:
            d_weights = d_out.new_empty(rows, dtype=torch.float32) if weights is None else torch.empty_like(weights)
        else:
            d_weights = d_out.new_zeros((rows,) if weights is None else weights.shape, dtype=torch.float32)
        if rows and columns:
            _done(ops.k3_moe_activation_backward(d_gate, d_up, scaled, d_weights, d_out, gate, up, weights, routes, offsets,
                                                 0 if offsets is None else offsets.shape[0] - 1, rows, columns, count,
                                                 self.activation, self.beta, self.linear_beta), "k3_moe_activation_backward")
        return d_gate, d_up, scaled, d_weights
