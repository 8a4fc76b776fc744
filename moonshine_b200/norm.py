"""RMS norm with the residual's addition and an 8-bit output, and its gradient (``include/k3_moe_norm.h``), on
torch tensors.

    before = norm.RmsNorm(weight, epsilon=1e-5)             # bf16 [hidden]
    r = before.forward(x, residual, y=False, codes=True)    # r.sum, r.codes, r.scales, r.rstd
    out = fp8.Fp8Linear(...).forward_codes(r.codes, r.scales)
    dx, d_weight = before.backward(dy, r.sum, r.rstd, d_sum)
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import ops
from .balance import _check
from .fp8 import _done, _matrix, _placed, _Workspace, pitch, scale_pitch

_TYPES = {torch.bfloat16: ops.NORM_BF16, torch.float32: ops.NORM_F32}


class Normed(NamedTuple):
    """What a forward pass leaves; what was not asked for is None."""
    sum: torch.Tensor                        # x + residual, x itself without one
    y: torch.Tensor | None                   # bf16 [rows, hidden]
    codes: torch.Tensor | None               # float8_e4m3fn [rows, pitch(hidden)]
    scales: torch.Tensor | None              # f32 [rows, scale_pitch(hidden)]
    rstd: torch.Tensor                       # f32 [rows]


class RmsNorm:
    """y = s rstd weight, s = x + residual, for ``weight`` bf16 [hidden].  x, the residual and their sum are bf16 or f32."""

    def __init__(self, weight: torch.Tensor, epsilon: float = 1e-5):
        if weight.dim() != 1 or weight.dtype is not torch.bfloat16 or not weight.is_contiguous():
            raise ValueError(f"weight: expected contiguous bfloat16 [hidden], got {weight.dtype} {list(weight.shape)}")
        self.weight, self._device, self.hidden, self.epsilon = weight, weight.device, weight.shape[0], float(epsilon)
        self._workspace = _Workspace(lambda rows: ops.k3_moe_norm_workspace_bytes(rows, self.hidden))

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None, y: bool = True, codes: bool = False) -> Normed:
        """x, residual [rows, hidden] -> their sum, the normalised rows in bf16 (``y``), in E4M3 (``codes``), or both."""
        rows, hidden = _matrix(x, "x", self.hidden, _TYPES)
        if residual is not None:
            _check(residual, "residual", x.dtype, (rows, hidden))
        if not (y or codes):
            raise ValueError("y and codes: one of them at least")
        _placed(("x", x), ("residual", residual), tables=self._device)
        # sizes one by one and empty_like: 1.3 to 1.5 us of the host's time each, new_empty of a tuple 1.9
        total = x if residual is None else torch.empty_like(x)
        out = torch.empty_like(x, dtype=torch.bfloat16) if y else None
        q = scales = None
        if codes:
            q = torch.empty(rows, pitch(hidden), dtype=torch.float8_e4m3fn, device=x.device)
            scales = torch.empty(rows, scale_pitch(hidden), dtype=torch.float32, device=x.device)
        rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
        if rows:
            _done(ops.k3_moe_norm(None if residual is None else total, out, q, scales, rstd, x, residual, self.weight, rows, hidden,
                                  _TYPES[x.dtype], self.epsilon), "k3_moe_norm")
        return Normed(total, out, q, scales, rstd)

    def backward(self, dy: torch.Tensor, sum: torch.Tensor, rstd: torch.Tensor, d_sum: torch.Tensor | None = None,
                 into: torch.Tensor | None = None):
        """dy bf16 [rows, hidden], the forward pass's sum and rstd, and d_sum [rows, hidden] of the sum's type, what its
        other readers send back -> the gradient by x and by the residual, of that type, and d_weight f32 [hidden], or
        added to ``into``."""
        rows, hidden = _matrix(sum, "sum", self.hidden, _TYPES)
        _check(dy, "dy", torch.bfloat16, (rows, hidden))
        _check(rstd, "rstd", torch.float32, (rows,))
        if d_sum is not None:
            _check(d_sum, "d_sum", sum.dtype, (rows, hidden))
        if into is not None:
            _check(into, "into", torch.float32, (hidden,))
        _placed(("dy", dy), ("sum", sum), ("rstd", rstd), ("d_sum", d_sum), ("into", into), tables=self._device)
        dx = torch.empty_like(sum)
        if rows == 0:
            return dx, into if into is not None else sum.new_zeros(hidden, dtype=torch.float32)
        d_weight = into if into is not None else sum.new_empty(hidden, dtype=torch.float32)
        ws = self._workspace.of(rows, sum.device)
        _done(ops.k3_moe_norm_backward(dx, d_weight, dy, sum, rstd, d_sum, self.weight, rows, hidden, _TYPES[sum.dtype],
                                       int(into is not None), ws, self._workspace.bytes), "k3_moe_norm_backward")
        return dx, d_weight
