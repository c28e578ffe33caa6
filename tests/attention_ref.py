"""The attention layer's operators in 64 bits on the CPU, written from their
formulas, for the tests; and what their roundings allow."""
import math

import torch

BF16 = torch.finfo(torch.bfloat16).eps / 2  # half a step, relative
F32 = torch.finfo(torch.float32).eps / 2


def paged_rows(pages, table, n):
    """Keys 0 .. n-1 of a sequence: [n, heads, D] in 64 bits; a page outside
    the cache holds zeros."""
    page = pages.shape[1]
    out = torch.zeros(n, pages.shape[2], pages.shape[3], dtype=torch.float64)
    for j in range(n):
        p = int(table[j // page])
        if 0 <= p < pages.shape[0]:
            out[j] = pages[p, j % page].double()
    return out


def attention(q, k_pages, v_pages, kv_len, table, q_start=None, prefix_pages=None, prefix_len=0,
              visible=None, scale=None, causal=True, window=0, softcap=0.0, slopes=None, gate=None):
    """Returns out, lse and the bound of their errors, all in 64 bits.

    bound of out: its rounding to bf16, and the rounding of each weight to
    bf16 before the second product, 2^-8 sum p |v| / sum p; fp32 sums and
    scores add `slack` to every exponent (see below), which moves the
    weights by that relative amount."""
    T, H, D = q.shape
    KV = k_pages.shape[2]
    G = H // KV
    scale = 1 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(T, H, D, dtype=torch.float64)
    tol = torch.zeros(T, H, D, dtype=torch.float64)
    lse = torch.full((T, H), -math.inf, dtype=torch.float64)
    lse_tol = torch.zeros(T, H, dtype=torch.float64)
    B = len(kv_len)
    for b in range(B):
        t0, t1 = (b, b + 1) if q_start is None else (int(q_start[b]), int(q_start[b + 1]))
        n, ql = min(int(kv_len[b]), table.shape[1] * k_pages.shape[1]), t1 - t0
        k, v = paged_rows(k_pages, table[b], n), paged_rows(v_pages, table[b], n)
        if prefix_len:
            k = torch.cat([paged_rows(k_pages, prefix_pages, prefix_len), k])
            v = torch.cat([paged_rows(v_pages, prefix_pages, prefix_len), v])
        N = prefix_len + n
        j = torch.arange(N)
        p = prefix_len + n - ql + torch.arange(ql)
        seen = torch.ones(ql, N, dtype=torch.bool)
        if causal:
            first = 0 if visible is None else int(visible[b])
            seen &= j[None] < torch.clamp(p + 1, min=first)[:, None]
        if window:
            seen &= j[None] > p[:, None] - window
        for h in range(H):
            x, kk, vv = q[t0:t1, h].double(), k[:, h // G], v[:, h // G]
            # Masked places may hold anything: they take no part.
            s = x @ torch.where(seen.any(0)[:, None], kk, 0.0).T * scale
            size = x.abs() @ torch.where(seen.any(0)[:, None], kk, 0.0).abs().T * abs(scale)
            if softcap:
                s = softcap * torch.tanh(s / softcap)
                size = size + softcap
            if slopes is not None:
                d = (p[:, None] - j[None]).abs().double()
                s = s - float(slopes[h]) * d
                size = size + abs(float(slopes[h])) * d
            s = torch.where(seen, s, -math.inf)
            some = seen.any(1)
            if not some.any():
                continue
            m = s.max(1, keepdim=True).values
            w = torch.where(some[:, None], torch.exp(s - torch.where(some[:, None], m, 0.0)), 0.0)
            l = w.sum(1, keepdim=True)
            vs = torch.where(seen.any(0)[:, None], vv, 0.0)
            w = w / torch.where(l > 0, l, 1.0)
            o, mag = w @ vs, w @ vs.abs()
            # fp32: a product sum of D terms, the scaling, the cap or bias and
            # the exponential (2 units), each 2^-24 of the terms' size; the
            # sums over keys (a few dozen partial sums per lane, 64 allowed).
            slack = (F32 * ((D + 16) * torch.where(seen, size, 0.0).max(1, keepdim=True).values + 64))
            o_tol = BF16 * mag + 2 * slack * mag
            if gate is not None:
                g = torch.sigmoid(gate[t0:t1, h].double())
                o, o_tol = o * g, o_tol * g
            out[t0:t1, h] = o
            tol[t0:t1, h] = BF16 * (o.abs() + o_tol) + o_tol + 1e-30
            lse[t0:t1, h] = torch.where(some, (m + torch.log(l))[:, 0], -math.inf)
            lse_tol[t0:t1, h] = (slack + 4 * F32 * (m.abs() + torch.log(l).abs()))[:, 0]
    return out, lse, tol, lse_tol


def head_norm(x, w, eps, offset):
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * (w.double() + offset)


def rotate(x, ang, interleaved, scale=1.0):
    """x [T, h, D], ang [T, R / 2], 64 bits."""
    half = ang.shape[1]
    i = torch.arange(half)
    e, o = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    c, s = torch.cos(ang)[:, None] * scale, torch.sin(ang)[:, None] * scale
    y = x.clone()
    y[..., e] = x[..., e] * c - x[..., o] * s
    y[..., o] = x[..., o] * c + x[..., e] * s
    return y


def check(got, ref, tol, what):
    got = got.double().cpu()
    same = torch.isfinite(ref)
    assert torch.equal(torch.isfinite(got), same), f"{what}: finite where it must not be, or not"
    assert torch.equal(got[~same & ~torch.isnan(ref)], ref[~same & ~torch.isnan(ref)]), what
    over = ((got - ref).abs() - tol)[same]
    if over.numel():
        worst = float(over.max())
        assert worst <= 0, f"{what}: {int((over > 0).sum())} of {over.numel()} beyond the bound, worst by {worst:.3g}"
