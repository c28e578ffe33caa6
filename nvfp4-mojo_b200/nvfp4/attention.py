"""Softmax attention over a paged key/value cache (include/nvfp4_attention.h):
`kv_append` (keys and values into the cache, heads normed and rotated on the
way) and `paged_attention` (prompts, single tokens, shared prefixes).

The handles (`PagedKVCache`, `AttentionBatch`, `AttentionConfig`, `Rotary`)
check their tensors once; a serving loop builds a batch per step and calls it
for every layer.  They keep their tensors alive and read no device memory.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from . import _lib

_byref = ctypes.byref
_DT = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}


_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


def _launch(t: torch.Tensor, stream, fn, *args) -> None:
    """fn(*args, stream) with t's device current; stream None: the current one
    of t's device.  Raises what fn reports."""
    dev = t.get_device()
    if stream is None:
        stream = _raw_stream(dev)
    elif isinstance(stream, torch.cuda.Stream):
        stream = stream.cuda_stream
    if dev == _current_device():
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, stream)
    if rc:
        _lib.check(rc)


def _new(t: torch.Tensor, stream, shape, dtype) -> torch.Tensor:
    """Memory on t's device that belongs to the stream of the call."""
    if stream is not None:
        if not isinstance(stream, torch.cuda.Stream):
            stream = torch.cuda.ExternalStream(int(stream), device=t.device)
        with torch.cuda.stream(stream):
            return torch.empty(shape, dtype=dtype, device=t.device)
    if t.dtype is dtype and t.shape == shape and t.is_contiguous():
        return torch.empty_like(t)
    return t.new_empty(shape, dtype=dtype)


def _check_device(t: torch.Tensor, **others) -> None:
    d = t.get_device()
    if d < 0:
        raise ValueError("tensors must be CUDA tensors (there is no CPU path)")
    for name, o in others.items():
        if o is not None and o.get_device() != d:
            raise ValueError(f"{name} must be a CUDA tensor on {t.device}")


def _i32(t: torch.Tensor, name: str, dim: int) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.dim() != dim:
        raise TypeError(f"{name} must be an int32 tensor of {dim} dimension(s)")
    if dim == 1 and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


def _int32(x, name: str) -> int:
    """x for an int32 field: ctypes would drop the bits beyond it."""
    x = int(x)
    if not -2 ** 31 <= x < 2 ** 31:
        raise ValueError(f"{name} {x} is out of range")
    return x


class PagedKVCache:
    """Keys and values in pages: k and v bf16 [num_pages, page_size,
    num_kv_heads, head_dim], any strides with contiguous heads (a permuted
    view of [num_pages, num_kv_heads, page_size, head_dim], or k and v as
    slices of one buffer)."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        if k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16:
            raise TypeError("the cache must be bf16")
        if k.dim() != 4 or v.shape != k.shape:
            raise ValueError("k and v must be [num_pages, page_size, num_kv_heads, head_dim]")
        if k.stride(3) != 1 or v.stride(3) != 1:
            raise ValueError("head rows must be contiguous")
        _check_device(k, v=v)
        self.k, self.v, self.device = k, v, k.get_device()
        n, self.page_size, self.num_kv_heads, self.head_dim = k.shape
        s = ctypes.c_int64 * 3
        self._c = _lib.KvCache(k.data_ptr(), v.data_ptr(), s(*k.stride()[:3]), s(*v.stride()[:3]),
                               n, self.page_size, self.num_kv_heads, self.head_dim)
        self._ref = ctypes.byref(self._c)

    @classmethod
    def empty(cls, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int,
              device="cuda") -> "PagedKVCache":
        shape = (num_pages, page_size, num_kv_heads, head_dim)
        return cls(torch.empty(shape, dtype=torch.bfloat16, device=device),
                   torch.empty(shape, dtype=torch.bfloat16, device=device))


class AttentionBatch:
    """One step's sequences.  kv_len int32 [B]: each sequence's keys, this
    step's tokens included; page_table int32 [B, max_pages] (one row expanded to
    B where all sequences have the same pages); q_start int32
    [B + 1]: the tokens of sequence b are rows q_start[b] : q_start[b + 1] of
    the call (None: one token per sequence), at most max_q_len each, num_tokens
    in all.  prefix_pages int32 and prefix_len: a prefix that every sequence
    shares and kv_len does not count.  visible_len int32 [B]: positions below
    it are seen by every query of the sequence, also by those before them (but
    no further back than a window reaches).

    Lengths and tables stay on the device and are read when the call runs, so
    a captured call can be replayed after they were rewritten in place."""

    def __init__(self, kv_len: torch.Tensor, page_table: torch.Tensor,
                 q_start: Optional[torch.Tensor] = None, num_tokens: Optional[int] = None,
                 max_q_len: int = 1, prefix_pages: Optional[torch.Tensor] = None,
                 prefix_len: int = 0, visible_len: Optional[torch.Tensor] = None):
        B = _i32(kv_len, "kv_len", 1).shape[0]
        _i32(page_table, "page_table", 2)
        if page_table.shape[0] != B or (page_table.shape[1] > 1 and page_table.stride(1) != 1):
            raise ValueError("page_table must be [num_seqs, max_pages] with contiguous rows")
        # The rows' distance means nothing for one row; 0 is one row expanded to all sequences.
        table_stride = page_table.stride(0) if B > 1 else page_table.shape[1]
        if 0 < table_stride < page_table.shape[1]:
            raise ValueError("page_table rows must not overlap")
        if q_start is None:
            if max_q_len != 1 or num_tokens not in (None, B):
                raise ValueError("without q_start every sequence has one token")
            num_tokens = B
        elif _i32(q_start, "q_start", 1).shape[0] != B + 1:
            raise ValueError("q_start must be [num_seqs + 1]")
        elif num_tokens is None:
            raise ValueError("q_start needs num_tokens (the rows of the call)")
        if (prefix_pages is None) != (prefix_len == 0):
            raise ValueError("prefix_pages and prefix_len go together")
        if prefix_pages is not None:
            _i32(prefix_pages, "prefix_pages", 1)
        if visible_len is not None and _i32(visible_len, "visible_len", 1).shape[0] != B:
            raise ValueError("visible_len must be [num_seqs]")
        _check_device(kv_len, page_table=page_table, q_start=q_start, prefix_pages=prefix_pages,
                      visible_len=visible_len)
        self.tensors = (kv_len, page_table, q_start, prefix_pages, visible_len)
        self.num_seqs, self.num_tokens, self.max_q_len = B, int(num_tokens), _int32(max_q_len, "max_q_len")
        self.prefix_len, self.device = _int32(prefix_len, "prefix_len"), kv_len.get_device()
        p = lambda t: None if t is None else t.data_ptr()
        self._c = _lib.AttnBatch(B, self.max_q_len, self.num_tokens, p(q_start), kv_len.data_ptr(),
                                 page_table.data_ptr(), table_stride, page_table.shape[1],
                                 self.prefix_len, p(prefix_pages), p(visible_len))
        self._ref = ctypes.byref(self._c)

    def _check_pages(self, page_size: int) -> None:
        pages = self.tensors[3]
        if pages is not None and pages.shape[0] * page_size < self.prefix_len:
            raise ValueError("prefix_pages hold fewer than prefix_len keys")


class AttentionConfig:
    """Heads and scores: s = scale * q.k (scale: 1 / sqrt(head_dim)), then
    softcap * tanh(s / softcap) where softcap > 0.  causal: a query sees the
    keys up to its own position; window > 0: only the last `window` of them."""

    def __init__(self, num_heads: int, num_kv_heads: int, head_dim: int,
                 scale: Optional[float] = None, causal: bool = True, window: int = 0,
                 softcap: float = 0.0):
        self.num_heads, self.num_kv_heads = _int32(num_heads, "num_heads"), _int32(num_kv_heads, "num_kv_heads")
        self.head_dim = _int32(head_dim, "head_dim")
        self._c = _lib.AttnDesc(self.num_heads, self.num_kv_heads, self.head_dim, int(bool(causal)),
                                _int32(window, "window"),
                                1.0 / math.sqrt(head_dim) if scale is None else scale, softcap)
        self._ref = ctypes.byref(self._c)


class Rotary:
    """Rotation of the first 2 * len(inv_freq) values of a head: pair i by
    position[axes[i]] * inv_freq[i] (fp32).  axes int32 (None: axis 0):
    which row of the positions turns the pair (time, height, width).  Pairs are
    (i, i + R / 2), or (2 i, 2 i + 1) when interleaved."""

    def __init__(self, inv_freq: torch.Tensor, axes: Optional[torch.Tensor] = None,
                 interleaved: bool = False, scale: float = 1.0):
        if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
            raise ValueError("inv_freq must be contiguous fp32 [rotary_dim / 2]")
        if axes is not None and _i32(axes, "axes", 1).shape != inv_freq.shape:
            raise ValueError("axes must be [rotary_dim / 2]")
        _check_device(inv_freq, axes=axes)
        self.tensors, self.device = (inv_freq, axes), inv_freq.get_device()
        self._c = _lib.RotaryDesc(inv_freq.data_ptr(), None if axes is None else axes.data_ptr(),
                                  2 * inv_freq.shape[0], int(interleaved), scale)
        self._ref = ctypes.byref(self._c)


def _head_rows(t: torch.Tensor, name: str, tokens: int, heads: int, dim: int) -> "_lib.HeadRows":
    if t.shape != (tokens, heads, dim):
        raise ValueError(f"{name} must be [{tokens}, {heads}, {dim}], not {list(t.shape)}")
    s = t.stride()
    if s[2] != 1:
        raise ValueError(f"{name} head rows must be contiguous")
    return _lib.HeadRows(t.data_ptr(), s[0], s[1])


def kv_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: PagedKVCache,
              batch: AttentionBatch, rotary: Optional[Rotary] = None,
              positions: Optional[torch.Tensor] = None, q_norm: Optional[torch.Tensor] = None,
              k_norm: Optional[torch.Tensor] = None, norm_eps: float = 1e-6,
              norm_offset: float = 0.0, q_out: Optional[torch.Tensor] = None,
              stream=None) -> torch.Tensor:
    """Appends this step's keys and values to the cache and returns the
    queries for `paged_attention`.

    q [T, num_heads, D], k and v [T, num_kv_heads, D]: bf16 or fp32, any token
    and head strides (slices of one projection).  q and k are RMS-normed per
    head where q_norm / k_norm (bf16 [D]) are given, then rotated.  positions
    int32 [T] or [axes, T] (one row expanded where the axes agree; None: the
    token's place in its sequence).  q_out bf16 [T, num_heads, D]; it may be q."""
    L = _lib.load()
    T, D = batch.num_tokens, cache.head_dim
    dtype = q.dtype
    if dtype not in _DT or k.dtype is not dtype or v.dtype is not dtype:
        raise TypeError("q, k and v must all be bf16 or all fp32")
    H = q.shape[1] if q.dim() == 3 else 0
    rq = _head_rows(q, "q", T, H, D)
    rk = _head_rows(k, "k", T, cache.num_kv_heads, D)
    rv = _head_rows(v, "v", T, cache.num_kv_heads, D)
    if q_out is None:
        q_out = _new(q, stream, (T, H, D), torch.bfloat16)
    elif q_out.dtype is not torch.bfloat16:
        raise TypeError("q_out must be bf16")
    ro = _head_rows(q_out, "q_out", T, H, D)
    dev = q.get_device()
    if dev < 0 or k.get_device() != dev or v.get_device() != dev or q_out.get_device() != dev or \
            cache.device != dev or batch.device != dev or \
            (rotary is not None and rotary.device != dev):
        raise ValueError("q, k, v, q_out, cache, batch and rotary must be on one CUDA device")
    pos, stride, axes = None, 0, 1
    if positions is not None:
        if positions.dtype is not torch.int32 or positions.dim() not in (1, 2) or \
                positions.shape[-1] != T or (T > 1 and positions.stride(-1) != 1):
            raise ValueError("positions must be int32 [T] or [axes, T] with contiguous rows")
        if positions.get_device() != dev:
            raise ValueError("positions must be on the tensors' device")
        pos = positions.data_ptr()
        if positions.dim() == 2:
            axes, stride = positions.shape[0], positions.stride(0)
            if axes > 1 and 0 < stride < T:
                raise ValueError("positions must not overlap from axis to axis")
    norm = None
    if q_norm is not None or k_norm is not None:
        for w, name in ((q_norm, "q_norm"), (k_norm, "k_norm")):
            if w is not None and (w.dtype is not torch.bfloat16 or w.shape != (D,) or
                                  not w.is_contiguous() or w.get_device() != dev):
                raise ValueError(f"{name} must be contiguous bf16 [head_dim] on the tensors' device")
        norm = _byref(_lib.QkNorm(None if q_norm is None else q_norm.data_ptr(),
                                  None if k_norm is None else k_norm.data_ptr(), norm_eps,
                                  norm_offset))
    _launch(q, stream, L.nvfp4_kv_append, cache._ref, batch._ref,
            None if rotary is None else rotary._ref, norm, _byref(rq), _byref(rk), _byref(rv),
            _DT[dtype], H, pos, stride, axes, _byref(ro))
    return q_out


def _workspace_bytes(config: AttentionConfig, batch: AttentionBatch, device) -> int:
    L = _lib.load()
    with torch.cuda.device(device):
        need = L.nvfp4_attention_workspace_size(config._ref, batch._ref)
    if need == 0:
        raise ValueError("unsupported attention: " + L.nvfp4_last_error_string().decode())
    return need


def attention_workspace(config: AttentionConfig, batch: AttentionBatch, device="cuda") -> torch.Tensor:
    """A workspace for `paged_attention` calls of this shape (or any smaller
    one: fewer tokens, a shorter max_q_len), one call at a time."""
    return torch.empty(_workspace_bytes(config, batch, device), dtype=torch.uint8, device=device)


def paged_attention(q: torch.Tensor, cache: PagedKVCache, batch: AttentionBatch,
                    config: AttentionConfig, slopes: Optional[torch.Tensor] = None,
                    gate: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                    return_lse: bool = False, workspace: Optional[torch.Tensor] = None,
                    stream=None):
    """softmax(scores) v of q [T, num_heads, D] (bf16) over each sequence's
    keys in the cache, times sigmoid(gate) where gate (bf16, like q) is given.

    slopes fp32 [num_heads]: subtracts slopes[h] * |distance| from the scores.
    Returns out [T, num_heads, D] bf16, or (out, lse) with lse fp32 [T,
    num_heads] the log-sum-exp of the scores.  A query that sees no key gets 0
    and -inf.  `workspace`: from `attention_workspace` (None: allocated)."""
    L = _lib.load()
    T, H, D = batch.num_tokens, config.num_heads, config.head_dim
    bf16 = torch.bfloat16
    if q.dtype is not bf16:
        raise TypeError("q must be bf16")
    rq = _head_rows(q, "q", T, H, D)
    if out is None:
        out = _new(q, stream, (T, H, D), bf16)
    lse = _new(q, stream, (T, H), torch.float32) if return_lse else None
    if workspace is None:
        workspace = _new(q, stream, _workspace_bytes(config, batch, q.get_device()), torch.uint8)
    if out.dtype is not bf16 or (gate is not None and gate.dtype is not bf16):
        raise TypeError("out and gate must be bf16")
    ro = _head_rows(out, "out", T, H, D)
    rg = None if gate is None else _byref(_head_rows(gate, "gate", T, H, D))
    if slopes is not None and (slopes.dtype is not torch.float32 or slopes.shape != (H,) or
                               not slopes.is_contiguous()):
        raise ValueError("slopes must be contiguous fp32 [num_heads]")
    if not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    if batch.prefix_len:
        batch._check_pages(cache.page_size)
    dev = q.get_device()
    if dev < 0 or out.get_device() != dev or workspace.get_device() != dev or \
            cache.device != dev or batch.device != dev or \
            (gate is not None and gate.get_device() != dev) or \
            (slopes is not None and slopes.get_device() != dev):
        raise ValueError("q, out, gate, slopes, workspace, cache and batch must be on one CUDA device")
    _launch(q, stream, L.nvfp4_paged_attention, config._ref, _byref(rq), cache._ref, batch._ref,
            None if slopes is None else slopes.data_ptr(), rg, _byref(ro),
            None if lse is None else lse.data_ptr(), workspace.data_ptr(), workspace.nbytes)
    return (out, lse) if return_lse else out


__all__ = ["PagedKVCache", "AttentionBatch", "AttentionConfig", "Rotary", "kv_append",
           "attention_workspace", "paged_attention"]
