"""The norms around a block with its gate and residual (include/nvfp4_norm.h)."""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib
from .attention import _call_stream, _check_device, _on_stream

_DT = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}
_ACT = {None: _lib.GATE_LINEAR, "linear": _lib.GATE_LINEAR, "sigmoid": _lib.GATE_SIGMOID}


def _rows(t: torch.Tensor, name: str, shape=None) -> torch.Tensor:
    if t.dtype not in _DT:
        raise TypeError(f"{name} must be bf16 or fp32")
    if t.dim() != 2 or (shape is not None and t.shape != shape):
        raise ValueError(f"{name} must be [rows, hidden]" + (f" = {tuple(shape)}" if shape else ""))
    if t.stride(1) != 1 and t.shape[1] > 1:
        raise ValueError(f"{name} rows must be contiguous")
    return t


def _weight(t: Optional[torch.Tensor], name: str, hidden: int) -> Optional[int]:
    if t is None:
        return None
    if t.dtype != torch.bfloat16 or t.shape != (hidden,) or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous bf16 [hidden]")
    return t.data_ptr()


def norm_residual(x: torch.Tensor, residual: Optional[torch.Tensor] = None,
                  pre_weight: Optional[torch.Tensor] = None,
                  post_weight: Optional[torch.Tensor] = None,
                  gate: Optional[torch.Tensor] = None, gate_act: Optional[str] = "sigmoid",
                  scale: float = 1.0, eps: float = 1e-6, weight_offset: float = 0.0,
                  residual_out: Optional[torch.Tensor] = None, y: Optional[torch.Tensor] = None,
                  y_dtype=torch.bfloat16, stream=None):
    """One launch for what lies between two blocks:

        u = rms(x) * (post_weight + weight_offset)     (x itself without post_weight)
        r = residual + scale * act(gate) * u
        y = rms(r) * (pre_weight + weight_offset)      (None without pre_weight)

    x [rows, hidden] is the block's output, `residual` the stream (bf16 or
    fp32; None: nothing is added), gate bf16 [rows, hidden], [1, hidden],
    [hidden] or [rows, 1] with act "sigmoid" or "linear", weights bf16
    [hidden].  Returns (r, y); r has the residual's dtype (x's without one).
    `residual_out` may be `residual` (update in place)."""
    L = _lib.load()
    _rows(x, "x")
    rows, hidden = x.shape
    if residual is not None:
        _rows(residual, "residual", x.shape)
    if gate_act not in _ACT:
        raise ValueError(f"gate_act {gate_act!r}: 'sigmoid', 'linear' or None")
    res_dtype = x.dtype if residual is None else residual.dtype
    if residual_out is None:
        with _on_stream(x, stream):
            residual_out = torch.empty((rows, hidden), dtype=res_dtype, device=x.device)
    elif _rows(residual_out, "residual_out", x.shape).dtype != res_dtype:
        raise TypeError("residual_out must have the residual's dtype")
    if pre_weight is None:
        if y is not None:
            raise ValueError("y needs pre_weight")
    elif y is None:
        if y_dtype not in _DT:
            raise TypeError("y_dtype must be bf16 or fp32")
        with _on_stream(x, stream):
            y = torch.empty((rows, hidden), dtype=y_dtype, device=x.device)
    else:
        _rows(y, "y", x.shape)
    gr = gc = 0
    if gate is not None:
        if gate.dtype != torch.bfloat16:
            raise TypeError("gate must be bf16")
        if gate.dim() == 1:
            gate = gate[None]
        if gate.dim() != 2 or gate.shape[0] not in (1, rows) or gate.shape[1] not in (1, hidden):
            raise ValueError("gate must be [rows, hidden], [1, hidden], [hidden] or [rows, 1]")
        if gate.shape[1] > 1 and gate.stride(1) != 1:
            raise ValueError("gate rows must be contiguous")
        gr = gate.stride(0) if gate.shape[0] > 1 else 0
        gc = 1 if gate.shape[1] > 1 else 0
    _check_device(x, residual=residual, pre_weight=pre_weight, post_weight=post_weight, gate=gate,
                  residual_out=residual_out, y=y)
    d = _lib.NormDesc(rows, hidden, _DT[x.dtype], _DT[res_dtype],
                      _DT[y.dtype] if y is not None else 0, _ACT[gate_act], scale, eps,
                      weight_offset, x.stride(0), 0 if residual is None else residual.stride(0),
                      residual_out.stride(0), 0 if y is None else y.stride(0), gr, gc)
    with _call_stream(x, stream) as st:
        rc = L.nvfp4_norm_residual(
            ctypes.byref(d), x.data_ptr(), None if residual is None else residual.data_ptr(),
            _weight(post_weight, "post_weight", hidden), None if gate is None else gate.data_ptr(),
            _weight(pre_weight, "pre_weight", hidden), residual_out.data_ptr(),
            None if y is None else y.data_ptr(), st)
    _lib.check(rc)
    return residual_out, y


__all__ = ["norm_residual"]
