"""Linear layers and routed experts on E4M3 tables with one f32 scale per 128 x 128 block
(``include/k3_moe_fp8.h``), on torch tensors.

Codes are ``torch.float8_e4m3fn`` with rows padded to 16 bytes (``pitch``); activations get one
scale per row and 128 columns, weights one per 128 x 128.  An object keeps its tables and a
workspace that grows with the largest call, so its calls have to be ordered (one stream, or
streams that wait for one another), as those of ``MoELayer``.  A workspace that a captured call
used stays with the object: a graph may be replayed after larger calls, while the object lives.
All tensors of a call lie on the current CUDA device.

    table, scales = fp8.quantize_blocks(weight)             # bf16 or f32 [rows, columns]
    y = fp8.Fp8Linear(table, scales, rows, columns).forward(x)
    grad = fp8.Fp8LinearGradient(*fp8.transpose_blocks(table, scales, rows, columns), rows, columns)
    dx, dw = grad.by_input(dy), grad.by_weight(dy, x)
    out = fp8.Fp8Experts(w1, s1, w3, s3, w2, s2, top_k=16).forward(x, ids, weights)
"""
from __future__ import annotations

import torch

from . import _native, ops

BLOCK = 128
_TYPES = {torch.bfloat16: ops.FP8_BF16, torch.float32: ops.FP8_F32}
_ACTIVATIONS = {"situ": ops.ACT_SITU, "swiglu": ops.ACT_SWIGLU}


def pitch(columns: int) -> int:
    """Bytes of a row of codes."""
    return (columns + 15) // 16 * 16


def blocks(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


def scale_pitch(columns: int) -> int:
    """Scales of a row of activations."""
    return (blocks(columns) + 3) // 4 * 4


def _done(ok: bool, name: str) -> None:
    if not ok:
        raise RuntimeError(name + " failed")


# the calls behind torch.cuda.current_device and is_current_stream_capturing, a fraction of their time
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", torch.cuda.is_current_stream_capturing)


def _placed(first, *others, tables: torch.device | None = None) -> None:
    """Refuses a (name, tensor) that the kernels cannot read: they run on the current device, and take addresses.
    None among the others is passed over.  ``tables``: the device that an object's tables are on."""
    name, t = first
    here = t.get_device()
    wrong = here < 0 or here != _current_device()
    if not wrong:
        for name, t in others:
            if t is not None and t.get_device() != here:
                wrong = True
                break
    if wrong:
        raise ValueError(f"{name}: expected a tensor on the current CUDA device, got one on {t.device}")
    if tables is not None and tables.index != here:
        raise ValueError(f"{first[0]}: on {first[1].device}, the tables are on {tables}")


def _matrix(x: torch.Tensor, name: str, columns: int | None = None, dtypes=(torch.bfloat16,)) -> tuple[int, int]:
    shape = x.shape
    if len(shape) != 2 or x.dtype not in dtypes or (columns is not None and shape[1] != columns):
        raise ValueError(f"{name}: expected [rows, {columns if columns is not None else 'columns'}] of "
                         f"{' or '.join(str(d) for d in dtypes)}, got {list(shape)} {x.dtype}")
    return shape


def _table(codes: torch.Tensor, scales: torch.Tensor, lead: tuple, rows: int, columns: int, name: str) -> torch.device:
    """Checks a table; its device."""
    if codes.dtype != torch.float8_e4m3fn or tuple(codes.shape) != (*lead, rows, pitch(columns)):
        raise ValueError(f"{name}: expected float8_e4m3fn {[*lead, rows, pitch(columns)]}, got {codes.dtype} {list(codes.shape)}")
    if scales.dtype != torch.float32 or tuple(scales.shape) != (*lead, blocks(rows), blocks(columns)):
        raise ValueError(f"{name}: expected float32 scales {[*lead, blocks(rows), blocks(columns)]}, got {scales.dtype} "
                         f"{list(scales.shape)}")
    if codes.device != scales.device:
        raise ValueError(f"{name}: codes on {codes.device}, scales on {scales.device}")
    return codes.device


def _quantized(name: str, x: torch.Tensor, codes_shape: tuple, scales_shape: tuple):
    codes = x.new_empty(codes_shape, dtype=torch.float8_e4m3fn)
    scales = x.new_empty(scales_shape, dtype=torch.float32)
    rows, columns = x.shape
    if rows and columns:
        _done(getattr(ops, name)(codes, scales, x, rows, columns, _TYPES[x.dtype]), name)
    return codes, scales


def quantize_rows(x: torch.Tensor):
    """bf16 or f32 [rows, columns] -> codes [rows, pitch(columns)], scales [rows, scale_pitch(columns)]."""
    rows, columns = _matrix(x, "x", dtypes=_TYPES)
    _placed(("x", x))
    return _quantized("k3_moe_fp8_quantize_rows", x, (rows, pitch(columns)), (rows, scale_pitch(columns)))


def quantize_columns(x: torch.Tensor):
    """The same of x transposed: codes [columns, pitch(rows)], scales [columns, scale_pitch(rows)]."""
    rows, columns = _matrix(x, "x", dtypes=_TYPES)
    _placed(("x", x))
    return _quantized("k3_moe_fp8_quantize_columns", x, (columns, pitch(rows)), (columns, scale_pitch(rows)))


def quantize_blocks(x: torch.Tensor):
    """A weight table: codes [rows, pitch(columns)], scales [blocks(rows), blocks(columns)]."""
    rows, columns = _matrix(x, "x", dtypes=_TYPES)
    _placed(("x", x))
    return _quantized("k3_moe_fp8_quantize_blocks", x, (rows, pitch(columns)), (blocks(rows), blocks(columns)))


def transpose_blocks(codes: torch.Tensor, scales: torch.Tensor, rows: int, columns: int):
    """The table of the transposed matrix, for the gradient by the input."""
    _table(codes, scales, (), rows, columns, "table")
    _placed(("table", codes))
    to = torch.empty((columns, pitch(rows)), dtype=torch.float8_e4m3fn, device=codes.device)
    to_scales = torch.empty((blocks(columns), blocks(rows)), dtype=torch.float32, device=codes.device)
    _done(ops.k3_moe_fp8_transpose_blocks(to, to_scales, codes, scales, rows, columns), "k3_moe_fp8_transpose_blocks")
    return to, to_scales


class _Workspace:
    """Device scratch of an object for the largest sizes (tokens, or tokens and sequences) it has seen;
    ``need(*sizes)`` gives the bytes.  A graph keeps the addresses of the calls that it captured, so what was
    handed out during a capture is never given back, while other scratch is when a larger call replaces it."""

    def __init__(self, need):
        self._need, self._held, self._sizes, self.bytes = need, None, (), 0
        self._last, self._captured = None, []

    def _keep(self) -> torch.Tensor:
        if _capturing() and not any(t is self._held for t in self._captured):
            self._captured.append(self._held)
        return self._held

    def of(self, *sizes_device) -> torch.Tensor:
        if sizes_device == self._last:
            return self._keep()
        *sizes, device = sizes_device
        if self._held is not None and self._held.device == device and all(map(int.__le__, sizes, self._sizes)):
            self._last = sizes_device
            return self._keep()
        sizes = [max(pair) for pair in zip(sizes, self._sizes)] if self._sizes else sizes
        need = self._need(*sizes)
        if need == 0:
            raise RuntimeError("the sizes of this call are not supported")
        if self._held is not None:              # the last call may still be running on this stream
            self._held.record_stream(torch.cuda.current_stream(self._held.device))
        self._held = torch.empty(need, dtype=torch.uint8, device=device)
        self._sizes, self._last, self.bytes = sizes, sizes_device, need
        return self._keep()


class Fp8Linear:
    """y = x W^T for a table of W [rows, columns]."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, rows: int, columns: int):
        self._device = _table(codes, scales, (), rows, columns, "table")
        self.codes, self.scales, self.rows, self.columns = codes, scales, rows, columns
        self._workspace = _Workspace(lambda tokens: ops.k3_moe_fp8_linear_workspace_bytes(tokens, columns))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        """x bf16 [tokens, columns] -> bf16 [tokens, rows]."""
        tokens, _ = _matrix(x, "x", self.columns)
        _placed(("x", x), tables=self._device)
        out = x.new_empty((tokens, self.rows))
        if tokens:
            ws = self._workspace.of(tokens, x.device)
            _done(ops.k3_moe_fp8_linear(out, x, self.codes, self.scales, tokens, self.rows, self.columns, ws, self._workspace.bytes),
                  "k3_moe_fp8_linear")
        return out


class Fp8LinearGradient:
    """The gradients of y = x W^T, W [rows, columns], from the table of W transposed (``transpose_blocks``)."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, rows: int, columns: int):
        self.rows, self.columns = rows, columns
        self._by_input = Fp8Linear(codes, scales, columns, rows)
        self._workspace = _Workspace(lambda tokens: ops.k3_moe_fp8_weight_gradient_workspace_bytes(tokens, rows, columns))

    def by_input(self, dy: torch.Tensor) -> torch.Tensor:
        """dy bf16 [tokens, rows] -> dx bf16 [tokens, columns]."""
        return self._by_input.forward(dy)

    def by_weight(self, dy: torch.Tensor, x: torch.Tensor, into: torch.Tensor | None = None) -> torch.Tensor:
        """dy bf16 [tokens, rows], x bf16 [tokens, columns] -> dw f32 [rows, columns], or added to ``into``."""
        tokens, _ = _matrix(dy, "dy", self.rows)
        if _matrix(x, "x", self.columns)[0] != tokens:
            raise ValueError("dy and x: different numbers of tokens")
        if into is not None:
            _matrix(into, "into", self.columns, (torch.float32,))
            if into.shape[0] != self.rows:
                raise ValueError(f"into: expected {[self.rows, self.columns]}, got {list(into.shape)}")
        _placed(("dy", dy), ("x", x), ("into", into))
        if tokens == 0:
            return into if into is not None else torch.zeros((self.rows, self.columns), dtype=torch.float32, device=dy.device)
        dw = into if into is not None else torch.empty((self.rows, self.columns), dtype=torch.float32, device=dy.device)
        ws = self._workspace.of(tokens, dy.device)
        _done(ops.k3_moe_fp8_weight_gradient(dw, dy, x, tokens, self.rows, self.columns, int(into is not None), ws,
                                             self._workspace.bytes), "k3_moe_fp8_weight_gradient")
        return dw


class Fp8Experts:
    """The routed experts of a layer on such tables: gate ``w1`` and up ``w3`` [experts, expert_hidden, hidden],
    down ``w2`` [experts, hidden, expert_hidden], each with scales per expert and 128 x 128 block."""

    def __init__(self, w1, w1_scales, w3, w3_scales, w2, w2_scales, top_k: int, activation: str = "swiglu",
                 beta: float = 4.0, linear_beta: float = 25.0):
        if w1.dim() != 3 or activation not in _ACTIVATIONS:
            raise ValueError("w1: expected [experts, expert_hidden, hidden], activation 'swiglu' or 'situ'")
        experts, expert_hidden, hidden = w1.shape
        self._device = w1.device
        for name, codes, scales, rows, columns in (("w1", w1, w1_scales, expert_hidden, hidden),
                                                   ("w3", w3, w3_scales, expert_hidden, hidden),
                                                   ("w2", w2, w2_scales, hidden, expert_hidden)):
            if _table(codes, scales, (experts,), rows, columns, name) != self._device:
                raise ValueError(f"{name}: on {codes.device}, w1 on {self._device}")
            if not (codes.is_contiguous() and scales.is_contiguous()):
                raise ValueError("operator arguments must be contiguous")
        self.hidden, self.top_k = hidden, top_k
        self.tables = (w1, w1_scales, w3, w3_scales, w2, w2_scales)
        self.desc = _native.Fp8ExpertsDesc(
            hidden=hidden, expert_hidden=expert_hidden, experts=experts, top_k=top_k, activation=_ACTIVATIONS[activation],
            beta=beta, linear_beta=linear_beta, w1=w1.data_ptr(), w1_scales=w1_scales.data_ptr(), w3=w3.data_ptr(),
            w3_scales=w3_scales.data_ptr(), w2=w2.data_ptr(), w2_scales=w2_scales.data_ptr())
        self._workspace = _Workspace(lambda tokens: ops.k3_moe_fp8_experts_workspace_bytes(self.desc, tokens))

    def forward(self, x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor,
                shared: torch.Tensor | None = None) -> torch.Tensor:
        """x bf16 [tokens, hidden], ids int32 and weights f32 [tokens, top_k] -> bf16 [tokens, hidden], plus
        ``shared`` (bf16, the shared expert's output) if given."""
        tokens, _ = _matrix(x, "x", self.hidden)
        for name, t, dtype in (("ids", ids, torch.int32), ("weights", weights, torch.float32)):
            if t.dtype is not dtype or t.shape != (tokens, self.top_k):
                raise ValueError(f"{name}: expected {dtype} {[tokens, self.top_k]}, got {t.dtype} {list(t.shape)}")
        if shared is not None and _matrix(shared, "shared", self.hidden)[0] != tokens:
            raise ValueError("shared: another number of tokens than x")
        _placed(("x", x), ("ids", ids), ("weights", weights), ("shared", shared), tables=self._device)
        out = x.new_empty((tokens, self.hidden))
        if tokens:
            ws = self._workspace.of(tokens, x.device)
            _done(ops.k3_moe_fp8_experts_forward(self.desc, out, x, ids, weights, shared, tokens, ws, self._workspace.bytes),
                  "k3_moe_fp8_experts_forward")
        return out
