"""The norms around a block with its gate and residual (include/nvfp4_norm.h)."""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib
from .attention import _launch, _new

_DT = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}
_ACT = {None: _lib.GATE_LINEAR, "linear": _lib.GATE_LINEAR, "sigmoid": _lib.GATE_SIGMOID}


def _rows(t: torch.Tensor, name: str, shape, dev: int) -> int:
    """The row stride of t [rows, hidden]."""
    if t.dtype not in _DT:
        raise TypeError(f"{name} must be bf16 or fp32")
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, not {list(t.shape)}")
    row, col = t.stride()
    if col != 1 and shape[1] > 1:
        raise ValueError(f"{name} rows must be contiguous")
    if t.get_device() != dev:
        raise ValueError(f"{name} must be on the device of x")
    return row


def _weight(t: Optional[torch.Tensor], name: str, hidden: int, dev: int) -> Optional[int]:
    if t is None:
        return None
    if t.dtype is not torch.bfloat16 or t.shape != (hidden,) or not t.is_contiguous() or \
            t.get_device() != dev:
        raise ValueError(f"{name} must be contiguous bf16 [hidden] on the device of x")
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
    shape, dev = x.shape, x.get_device()
    if len(shape) != 2 or shape[1] > 32768:
        raise ValueError("x must be [rows, hidden], hidden at most 32768")
    if dev < 0:
        raise ValueError("x must be a CUDA tensor (there is no CPU path)")
    rows, hidden = shape
    xs = _rows(x, "x", shape, dev)
    rs = 0 if residual is None else _rows(residual, "residual", shape, dev)
    if gate_act not in _ACT:
        raise ValueError(f"gate_act {gate_act!r}: 'sigmoid', 'linear' or None")
    stream_like = x if residual is None else residual
    res_dtype = stream_like.dtype
    if residual_out is None:
        residual_out = _new(stream_like, stream, shape, res_dtype)
    elif residual_out.dtype is not res_dtype:
        raise TypeError("residual_out must have the residual's dtype")
    ros = _rows(residual_out, "residual_out", shape, dev)
    ys = 0
    if pre_weight is not None:
        if y is None:
            if y_dtype not in _DT:
                raise TypeError("y_dtype must be bf16 or fp32")
            y = _new(x, stream, shape, y_dtype)
        ys = _rows(y, "y", shape, dev)
    elif y is not None:
        raise ValueError("y needs pre_weight")
    gr = gc = 0
    if gate is not None:
        if gate.dtype is not torch.bfloat16 or gate.get_device() != dev:
            raise TypeError("gate must be bf16 on the device of x")
        if gate.dim() == 1:
            gate = gate[None]
        if gate.dim() != 2 or gate.shape[0] not in (1, rows) or gate.shape[1] not in (1, hidden):
            raise ValueError("gate must be [rows, hidden], [1, hidden], [hidden] or [rows, 1]")
        if gate.shape[1] > 1 and gate.stride(1) != 1:
            raise ValueError("gate rows must be contiguous")
        gr = gate.stride(0) if gate.shape[0] > 1 else 0
        gc = 1 if gate.shape[1] > 1 else 0
    d = _lib.NormDesc(rows, hidden, _DT[x.dtype], _DT[res_dtype], 0 if y is None else _DT[y.dtype],
                      _ACT[gate_act], scale, eps, weight_offset, xs, rs, ros, ys, gr, gc)
    _launch(x, stream, L.nvfp4_norm_residual, ctypes.byref(d), x.data_ptr(),
            None if residual is None else residual.data_ptr(),
            _weight(post_weight, "post_weight", hidden, dev),
            None if gate is None else gate.data_ptr(),
            _weight(pre_weight, "pre_weight", hidden, dev), residual_out.data_ptr(),
            None if y is None else y.data_ptr())
    return residual_out, y


__all__ = ["norm_residual"]
