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

``RoutedExperts`` is all of it for one layer: dispatch, products, activation and weighted sum, and their gradients.
"""
from __future__ import annotations

from typing import NamedTuple

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
            to = torch.empty(rows, columns, dtype=dtype, device=x.device)
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
            to = torch.empty(*shape, dtype=dtype, device=dy.device)
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

        Row r belongs to route ``routes[r]`` (int32 [rows], no route twice; None: route r), whose routing weight is
        that element of ``weights`` (f32, [tokens, top_k] say; None: 1 for each row).  ``d_out`` is the gradient that the
        down matrix sends back for the unweighted row; ``scaled``, weight times activation, is what that matrix's own
        gradient reads.  d_weights f32 has the shape of ``weights``, [rows] without them, and is 0
        for a route without a row; a row whose route is past the weights has weight 0.  With ``offsets`` rows outside of
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
        # zeros for routes that no row has, which only a table of routes can leave out (4 us of the host's time)
        whole = routes is None and offsets is None and rows and columns
        if weights is None:
            d_weights = (torch.empty if whole else torch.zeros)(rows, dtype=torch.float32, device=d_out.device)
        else:
            d_weights = torch.empty_like(weights) if whole else torch.zeros_like(weights)
        if rows and columns:
            _done(ops.k3_moe_activation_backward(d_gate, d_up, scaled, d_weights, d_out, gate, up, weights, routes, offsets,
                                                 0 if offsets is None else offsets.shape[0] - 1, rows, columns, count,
                                                 self.activation, self.beta, self.linear_beta), "k3_moe_activation_backward")
        return d_gate, d_up, scaled, d_weights


class Routed(NamedTuple):
    """What a forward pass of ``RoutedExperts`` leaves for the backward pass: the dispatch, and the rows it grouped."""
    offsets: torch.Tensor                    # int32 [experts + 1]
    routes: torch.Tensor                     # int32 [rows]: the route token * top_k + rank of a row
    tokens: torch.Tensor                     # int32 [rows]: its token
    place: torch.Tensor                      # int32 [tokens * top_k]: the row of a route, -1 where it has none
    weights: torch.Tensor
    x: torch.Tensor                          # bf16 [rows, hidden]
    gate: torch.Tensor                       # bf16 [rows, expert_hidden]
    up: torch.Tensor


class ExpertGradients(NamedTuple):
    x: torch.Tensor                          # bf16 [tokens, hidden]
    weights: torch.Tensor                    # f32 [tokens, top_k], for ``balance.RouterBalance.backward``
    w1: torch.Tensor                         # f32, as the matrices
    w3: torch.Tensor
    w2: torch.Tensor


class RoutedExperts:
    """The routed experts of a layer in bf16: gate ``w1`` and up ``w3`` [experts, expert_hidden, hidden], down ``w2``
    [experts, hidden, expert_hidden], hidden a multiple of 8.  The products' results are rounded to bf16, as are the rows' gradients; the
    gradient by x adds those of gate and up in f32 before its rounding.  Neither pass waits for the GPU."""

    def __init__(self, w1: torch.Tensor, w3: torch.Tensor, w2: torch.Tensor, top_k: int, activation: str = "swiglu",
                 beta: float = 4.0, linear_beta: float = 25.0):
        self.gate, self.up, self.down = GroupedProduct(w1), GroupedProduct(w3), GroupedProduct(w2)
        experts, expert_hidden, hidden = w1.shape
        if w3.shape != w1.shape or w2.shape != (experts, hidden, expert_hidden):
            raise ValueError(f"w1, w3 and w2: expected {list(w1.shape)} twice and {[experts, hidden, expert_hidden]}, got {list(w3.shape)} and "
                             f"{list(w2.shape)}")
        if hidden % 8:
            raise ValueError(f"w1: expected a multiple of 8 columns, which the weighted sum wants, got {hidden}")
        if not 0 < top_k <= min(experts, 32):
            raise ValueError(f"top_k: 1 to {min(experts, 32)}, got {top_k}")
        self.experts, self.hidden, self.expert_hidden, self.top_k = experts, hidden, expert_hidden, top_k
        self.activation = GatedActivation(activation, beta, linear_beta)
        self._by_w1, self._by_w3 = (GroupedWeightGradient(experts, expert_hidden, hidden) for _ in range(2))
        self._by_w2 = GroupedWeightGradient(experts, hidden, expert_hidden)
        self._workspace = _Workspace(lambda tokens: ops.k3_moe_dispatch_workspace_bytes(tokens, top_k, experts))

    def _gather(self, x, tokens):
        rows = x.new_empty((tokens.shape[0], self.hidden))
        _done(ops.k3_rocm_gather_rows_bf16(rows, x, tokens, tokens.shape[0], self.hidden), "k3_rocm_gather_rows_bf16")
        return rows

    def _combine(self, rows, place, weights):
        out = rows.new_empty((weights.shape[0], self.hidden))
        _done(ops.k3_moe_combine(out, rows, place, weights, None, weights.shape[0], self.top_k, self.hidden), "k3_moe_combine")
        return out

    def forward(self, x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor) -> tuple[torch.Tensor, Routed]:
        """x bf16 [tokens, hidden], ids int32 and weights f32 [tokens, top_k], as ``k3_moe_route`` writes them -> bf16
        [tokens, hidden], and what ``backward`` reads.  An id that is no expert's adds nothing and has no gradients; it
        raises bit 1 of ``k3_moe_device_status``."""
        tokens, _ = _matrix(x, "x", self.hidden)
        _check(ids, "ids", torch.int32, (tokens, self.top_k))
        _check(weights, "weights", torch.float32, (tokens, self.top_k))
        _placed(("x", x), ("ids", ids), ("weights", weights), tables=self.gate._device)
        rows = tokens * self.top_k
        # what a dispatch leaves out (an id that is no expert's): zeros stay an index inside, a place of -1 adds nothing
        offsets, routes, of_row = (ids.new_zeros(n) for n in (self.experts + 1, rows, rows))
        place = ids.new_full((rows,), -1)
        if tokens == 0:
            nothing = x.new_empty((0, self.expert_hidden))
            return x.new_empty((0, self.hidden)), Routed(offsets, routes, of_row, place, weights, x, nothing, nothing)
        ws = self._workspace.of(tokens, x.device)
        _done(ops.k3_moe_dispatch_build(offsets, routes, of_row, place, ids, tokens, self.top_k, self.experts, ws, self._workspace.bytes),
              "k3_moe_dispatch_build")
        x_rows = self._gather(x, of_row)
        gate, up = self.gate.forward(x_rows, offsets), self.up.forward(x_rows, offsets)
        out = self._combine(self.down.forward(self.activation.forward(gate, up), offsets), place, weights)
        return out, Routed(offsets, routes, of_row, place, weights, x_rows, gate, up)

    def backward(self, d_out: torch.Tensor, saved: Routed) -> ExpertGradients:
        """d_out bf16 [tokens, hidden] and what ``forward`` left -> the gradients by x, the routing weights and the matrices."""
        tokens, _ = _matrix(d_out, "d_out", self.hidden)
        if saved.weights.shape[0] != tokens:
            raise ValueError(f"d_out: expected {saved.weights.shape[0]} tokens, got {tokens}")
        _placed(("d_out", d_out), tables=self.gate._device)
        offsets = saved.offsets
        if tokens == 0:
            d_gate = d_up = scaled = saved.gate
            dx, d_rows, d_weights = d_out, d_out, torch.empty_like(saved.weights)
        else:
            d_rows = self._gather(d_out, saved.tokens)
            d_gate, d_up, scaled, d_weights = self.activation.backward(self.down.by_input(d_rows, offsets), saved.gate, saved.up,
                                                                       saved.weights, saved.routes, offsets)
            by_rows = self.gate.by_input(d_gate, offsets, dtype=torch.float32)
            self.up.by_input(d_up, offsets, into=by_rows)
            dx = self._combine(by_rows.to(torch.bfloat16), saved.place, torch.ones_like(saved.weights))
        return ExpertGradients(dx, d_weights, self._by_w1.forward(d_gate, saved.x, offsets), self._by_w3.forward(d_up, saved.x, offsets),
                               self._by_w2.forward(d_rows, scaled, offsets))
