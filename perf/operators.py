"""Measured work of the softmax-attention operators: appending to a paged
key/value cache with the rotation on the way, attention over that cache (for
prompts, for single tokens, and for a batch that shares a long prefix), and
the norms around a block with its gate and residual.

`own` False: the operators in plain torch operations, 32-bit arithmetic.
`own` True: the package's entry points (nvfp4.attention, nvfp4.norm).
"""
import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

# Head layouts (query heads, key/value heads, head size): the two models the
# package's loader and MoE configurations name, a multi-head layout and one
# with an odd number of query heads per key/value head.
LAYOUTS = [(32, 4, 128), (16, 2, 256), (8, 8, 64), (28, 4, 128), (16, 16, 128)]

_NORM = dict(kind="norm", tokens=1, hidden=2048, x32=False, r32=False, post=False, gate="none",
             scale=1.0, offset=0.0)
_APPEND = dict(kind="append", seqs=1, q_min=1, q_max=1, ctx_min=0, ctx_max=1000, heads=32, kv_heads=4,
               dim=128, page=64, rotary=128, axes=1, interleaved=False, norm=True, x32=False,
               first=0)
_ATTN = dict(kind="attention", seqs=1, q_min=1, q_max=1, ctx_min=0, ctx_max=1000, heads=32, kv_heads=4,
             dim=128, page=64, causal=True, window=0, softcap=0.0, slopes=False, visible=0,
             gate=False, prefix=0, lse=False)


def listed():
    return [
        # The norm before a block in a decode step of one sequence: the residual add and the norm.
        dict(_NORM, name="norm_token"),
        # A long prompt through a block with norms on both sides, an fp32 residual stream and a
        # sigmoid gate per token (a shared expert's).
        dict(_NORM, name="norm_prompt", tokens=16384, r32=True, post=True, gate="token", scale=0.5,
             offset=1.0),
        # A decode step of a batch: one new token per sequence.
        dict(_APPEND, name="append_tokens", seqs=64, ctx_max=2000, first=100000),
        # Prompts with images: three position axes, a quarter of the head rotated.
        dict(_APPEND, name="append_prompt", seqs=5, q_min=500, q_max=2500, ctx_max=40, heads=16,
             kv_heads=2, dim=256, page=16, rotary=64, axes=3),
        # One sequence being decoded, early in its answer.
        dict(_ATTN, name="token_one", ctx_min=600, ctx_max=700),
        # A serving batch of ragged contexts.
        dict(_ATTN, name="token_batch", seqs=64, ctx_min=200, ctx_max=12000),
        # Long contexts at head size 256 with the attention output gate, log-sum-exp returned.
        dict(_ATTN, name="token_long", seqs=6, ctx_min=9000, ctx_max=60000, heads=16, kv_heads=2,
             dim=256, page=16, gate=True, lse=True),
        # One long prompt.
        dict(_ATTN, name="prompt_long", q_min=8000, q_max=8192, ctx_max=0),
        # Ragged prompts that continue cached contexts, at head size 256.
        dict(_ATTN, name="prompt_ragged", seqs=4, q_min=301, q_max=1700, ctx_max=2001, heads=16,
             kv_heads=2, dim=256, page=16, gate=True),
        # Capped scores, a distance bias, a sliding window and an image prefix that sees itself.
        dict(_ATTN, name="prompt_capped", seqs=3, q_min=900, q_max=2100, ctx_max=100, heads=28,
             window=1024, softcap=50.0, slopes=True, visible=257),
        # Decoding for many users that share a long system prompt.
        dict(_ATTN, name="prefix_tokens", seqs=96, ctx_min=10, ctx_max=400, prefix=16384),
        # Their questions after that prompt, all at once.
        dict(_ATTN, name="prefix_prompt", seqs=8, q_min=40, q_max=130, ctx_max=0, heads=16,
             kv_heads=2, dim=256, prefix=8000, lse=True),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["norm", "append", "token", "token", "prompt", "prompt", "prefix"])
    if kind == "norm":
        hidden = rng.choice([1, 8]) * _spread(rng, 64, 1000)
        return dict(_NORM, tokens=_spread(rng, 1, 16384 * 2048 // max(hidden, 2048)), hidden=hidden,
                    x32=rng.random() < 0.3, r32=rng.random() < 0.5, post=rng.random() < 0.5,
                    gate=rng.choice(["none", "token", "channel", "full"]),
                    scale=rng.choice([1.0, 0.5]), offset=rng.choice([0.0, 1.0]))
    H, KV, D = rng.choice(LAYOUTS)
    page = rng.choice([16, 32, 64, 128])
    if kind == "append":
        many = rng.random() < 0.5
        return dict(_APPEND, seqs=_spread(rng, 1, 5 if many else 64), q_min=1,
                    q_max=_spread(rng, 2, 2400) if many else 1, ctx_max=_spread(rng, 1, 1000),
                    heads=H, kv_heads=KV, dim=D, page=page, rotary=rng.choice([D, D // 2, D // 4]),
                    axes=rng.choice([1, 3]), interleaved=rng.random() < 0.5,
                    norm=rng.random() < 0.5, x32=rng.random() < 0.3,
                    first=rng.choice([0, 0, 1000000]))
    opts = dict(heads=H, kv_heads=KV, dim=D, page=page, lse=rng.random() < 0.5,
                gate=rng.random() < 0.3, softcap=rng.choice([0.0, 0.0, 20.0, 50.0]),
                slopes=rng.random() < 0.2, window=rng.choice([0, 0, _spread(rng, 16, 4096)]))
    if kind == "token":
        seqs = _spread(rng, 1, 64)
        return dict(_ATTN, **{**opts, "seqs": seqs, "q_max": rng.choice([1, 1, 1, 4]),
                              "ctx_max": _spread(rng, 4, min(60000, 280000 // seqs))})
    if kind == "prompt":
        seqs = _spread(rng, 1, 4)
        return dict(_ATTN, **{**opts, "seqs": seqs, "q_min": 1, "q_max": _spread(rng, 17, 3900 // seqs),
                              "ctx_max": rng.choice([0, _spread(rng, 1, 1500)]),
                              "causal": rng.random() < 0.8,
                              "visible": rng.choice([0, 0, _spread(rng, 1, 500)])})
    return dict(_ATTN, **{**opts, "seqs": _spread(rng, 2, 48), "q_max": rng.choice([1, 1, 3]),
                          "ctx_max": _spread(rng, 4, 400), "prefix": _spread(rng, 100, 8192),
                          "window": 0})


def _lengths(c):
    """Queries and cached keys per sequence: ragged, the same for every seed."""
    r = random.Random(1000003 * c["seqs"] + 31 * c["q_max"] + c["ctx_max"])
    q = [r.randint(c["q_min"], c["q_max"]) for _ in range(c["seqs"])]
    ctx = [r.randint(c["ctx_min"], c["ctx_max"]) for _ in range(c["seqs"])]
    q[0], ctx[-1] = c["q_max"], c["ctx_max"]
    return q, [a + b for a, b in zip(q, ctx)]


def _intervals(c):
    """Per sequence the first key and the end of the keys that each of its queries sees."""
    P = c["prefix"]
    got = []
    for q, n in zip(*_lengths(c)):
        p = P + n - q + np.arange(q, dtype=np.int64)
        hi = np.maximum(p + 1, min(c["visible"], n)) if c["causal"] else np.full(q, P + n)
        lo = np.maximum(p - c["window"] + 1, 0) if c["window"] else np.zeros(q, np.int64)
        got.append((lo, np.maximum(np.minimum(hi, P + n), lo)))
    return got


def work(c):
    if c["kind"] == "norm":
        n, b = c["tokens"] * c["hidden"], 0
        b += n * (4 if c["x32"] else 2) + 2 * n * (4 if c["r32"] else 2) + 2 * n
        b += {"none": 0, "token": 2 * c["tokens"], "channel": 2 * c["hidden"], "full": 2 * n}[c["gate"]]
        return {"bytes": b + (2 if c["post"] else 1) * 2 * c["hidden"], "flops": 10 * n}
    T = sum(_lengths(c)[0])
    row = c["dim"] * 2
    if c["kind"] == "append":
        values = T * (c["heads"] + 2 * c["kv_heads"]) * c["dim"]
        return {"bytes": values * ((4 if c["x32"] else 2) + 2), "flops": 10 * values}
    seen = _intervals(c)
    keys = sum(int(hi.max() - max(lo.min(), c["prefix"])) for lo, hi in seen if hi.max() > lo.min())
    first = min(int(lo.min()) for lo, _ in seen)
    keys += max(0, c["prefix"] - first)
    pairs = sum(int((hi - lo).sum()) for lo, hi in seen)
    return {"bytes": keys * c["kv_heads"] * 2 * row + T * c["heads"] * row * (3 if c["gate"] else 2)
            + (4 * T * c["heads"] if c["lse"] else 0),
            "flops": 4 * pairs * c["heads"] * c["dim"]}


def _package():
    at = str(Path(__file__).resolve().parents[1] / "nvfp4-mojo_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import nvfp4.attention
    import nvfp4.norm

    return nvfp4.attention, nvfp4.norm


def _norm_inputs(c, g):
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")
    T, H = c["tokens"], c["hidden"]
    s = dict(x=n(T, H).to(torch.float32 if c["x32"] else torch.bfloat16),
             residual=(3.0 * n(T, H)).to(torch.float32 if c["r32"] else torch.bfloat16),
             pre=(1.0 - c["offset"] + 0.2 * n(H)).to(torch.bfloat16), post_w=None, gate=None)
    if c["post"]:
        s["post_w"] = (1.0 - c["offset"] + 0.2 * n(H)).to(torch.bfloat16)
    if c["gate"] != "none":
        shape = {"token": (T, 1), "channel": (1, H), "full": (T, H)}[c["gate"]]
        s["gate"] = n(*shape).to(torch.bfloat16)
    return s


def _paged(c, g):
    """Lengths, a shuffled page table and caches filled as by earlier steps."""
    q, n = _lengths(c)
    page, B = c["page"], c["seqs"]
    own_pages = [-(-k // page) for k in n]
    P = c.get("prefix", 0)
    P_pages = -(-P // page)
    total = sum(own_pages) + P_pages + 3
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    width = max(own_pages)
    starts = np.concatenate([[0], np.cumsum(own_pages)])[:B]
    at = torch.from_numpy(starts).cuda()[:, None] + torch.arange(width, device="cuda")[None]
    table = order[(P_pages + at).clamp(max=total - 1)].contiguous()
    shape = (total, page, c["kv_heads"], c["dim"])
    s = dict(k=torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16),
             v=torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16),
             table=table, prefix_pages=order[:P_pages].clone(),
             kv_len=torch.tensor(n, dtype=torch.int32, device="cuda"),
             q_start=torch.tensor(np.concatenate([[0], np.cumsum(q)]), dtype=torch.int32, device="cuda"),
             T=sum(q), q_max=max(q), kv_max=max(n))
    return s


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    if c["kind"] == "norm":
        s = _norm_inputs(c, g)
    else:
        s = _paged(c, g)
        T, H, KV, D = s["T"], c["heads"], c["kv_heads"], c["dim"]
        if c["kind"] == "append":
            # One projection's output, the heads' rows side by side.
            s["qkv"] = torch.randn(T, H + 2 * KV, D, generator=g, device="cuda").to(
                torch.float32 if c["x32"] else torch.bfloat16)
            half = c["rotary"] // 2
            s["inv_freq"] = (1e6 ** (-torch.arange(half, dtype=torch.float64) / half)).float().cuda()
            s["axis"] = (torch.arange(half) % c["axes"]).to(torch.int32).cuda()
            b = torch.repeat_interleave(torch.arange(c["seqs"], device="cuda"),
                                        (s["q_start"][1:] - s["q_start"][:-1]).long())
            s["seq"] = b
            s["at"] = s["kv_len"][b].long() - s["q_start"][b + 1] + torch.arange(T, device="cuda")
            # Time runs on with the text (from `first`, where a prefix came before); an image's
            # rows and columns start again.
            pos = torch.stack([c["first"] + s["at"], s["at"] % 61, (s["at"] * 7) % 53])[:c["axes"]]
            s["pos"] = pos.to(torch.int32).contiguous()
            s["qw"] = s["kw"] = None
            if c["norm"]:
                s["qw"] = (1 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(torch.bfloat16)
                s["kw"] = (1 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(torch.bfloat16)
        else:
            s["q"] = (2.0 * torch.randn(T, H, D, generator=g, device="cuda")).to(torch.bfloat16)
            s["gate"] = torch.randn(T, H, D, generator=g, device="cuda").to(torch.bfloat16) if c["gate"] else None
            s["slopes"] = (2.0 ** (-8.0 * (torch.arange(H, device="cuda") + 1) / H)).float() if c["slopes"] else None
            s["visible"] = torch.minimum(s["kv_len"], torch.tensor(c["visible"], dtype=torch.int32, device="cuda")) if c["visible"] else None
    s["c"] = c
    if own:  # the handles and workspace that a serving loop keeps over its layers
        A, N = s["package"] = _package()
        if c["kind"] != "norm":
            s["cache"] = A.PagedKVCache(s["k"], s["v"])
            s["batch"] = A.AttentionBatch(
                s["kv_len"], s["table"], q_start=None if s["q_max"] == 1 else s["q_start"],
                num_tokens=s["T"], max_q_len=s["q_max"], prefix_len=c.get("prefix", 0),
                prefix_pages=s["prefix_pages"] if c.get("prefix") else None,
                visible_len=s.get("visible"))
        if c["kind"] == "append":
            s["rotary"] = A.Rotary(s["inv_freq"], axes=s["axis"] if c["axes"] > 1 else None,
                                   interleaved=c["interleaved"])
        if c["kind"] == "attention":
            s["config"] = A.AttentionConfig(c["heads"], c["kv_heads"], c["dim"], causal=c["causal"],
                                            window=c["window"], softcap=c["softcap"])
            s["ws"] = A.attention_workspace(s["config"], s["batch"], device=s["q"].device)
    return s


def _run_own(s):
    A, N = s["package"]
    c = s["c"]
    if c["kind"] == "norm":
        r, y = N.norm_residual(s["x"], s["residual"], pre_weight=s["pre"], post_weight=s["post_w"],
                               gate=s["gate"], gate_act="sigmoid", scale=c["scale"],
                               weight_offset=c["offset"])
        return {"residual": r, "y": y}
    if c["kind"] == "append":
        H, KV = c["heads"], c["kv_heads"]
        q, k, v = s["qkv"].split([H, KV, KV], dim=1)
        q_out = A.kv_append(q, k, v, s["cache"], s["batch"], rotary=s["rotary"], positions=s["pos"],
                            q_norm=s["qw"], k_norm=s["kw"])
        return {"q": q_out, "k": s["k"], "v": s["v"]}
    out = A.paged_attention(s["q"], s["cache"], s["batch"], s["config"], slopes=s["slopes"],
                            gate=s["gate"], return_lse=c["lse"], workspace=s["ws"])
    return {"out": out[0], "lse": out[1]} if c["lse"] else {"out": out}


def _rms(x, w, offset):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * (w.float() + offset)


def _run_norm(s):
    c = s["c"]
    u = s["x"].float()
    if s["post_w"] is not None:
        u = _rms(u, s["post_w"], c["offset"])
    if s["gate"] is not None:
        u = u / (1 + torch.exp(-s["gate"].float()))
    r = s["residual"].float() + c["scale"] * u
    return {"residual": r.to(s["residual"].dtype), "y": _rms(r, s["pre"], c["offset"]).to(torch.bfloat16)}


def _rotate(x, ang, interleaved):
    """x [T, h, D] float, ang [T, R/2] in 64 bits."""
    half = ang.shape[1]
    cos, sin = ang.cos().float()[:, None], ang.sin().float()[:, None]
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else (x[..., :half], x[..., half:2 * half])
    u, w = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([u, w], -1).flatten(-2) if interleaved else torch.cat([u, w], -1)
    return torch.cat([turned, x[..., 2 * half:]], -1)


def _run_append(s):
    c = s["c"]
    H, KV = c["heads"], c["kv_heads"]
    x = s["qkv"].float()
    ang = (s["pos"][s["axis"].long()].double() * s["inv_freq"].double()[:, None]).t()
    q, k, v = x.split([H, KV, KV], dim=1)
    if c["norm"]:
        q, k = _rms(q, s["qw"], 0.0), _rms(k, s["kw"], 0.0)
    q, k = _rotate(q, ang, c["interleaved"]), _rotate(k, ang, c["interleaved"])
    page = s["table"][s["seq"], s["at"] // c["page"]].long()
    s["k"][page, s["at"] % c["page"]] = k.to(torch.bfloat16)
    s["v"][page, s["at"] % c["page"]] = v.to(torch.bfloat16)
    return {"q": q.to(torch.bfloat16), "k": s["k"], "v": s["v"]}


def _run_attention(s):
    c = s["c"]
    B, H, KV, D, P = c["seqs"], c["heads"], c["kv_heads"], c["dim"], c["prefix"]
    G, Lq, Lk = H // KV, s["q_max"], s["kv_max"]
    q_len = s["q_start"][1:] - s["q_start"][:-1]
    i = torch.arange(Lq, device="cuda")
    token = (s["q_start"][:-1, None] + i).clamp(max=s["T"] - 1).long()
    q = s["q"].float()[token].view(B, Lq, KV, G, D)
    pages = s["table"][:, :-(-Lk // c["page"])].long()
    k, v = (x[pages].view(B, -1, KV, D)[:, :Lk].float() for x in (s["k"], s["v"]))
    if P:
        pp = s["prefix_pages"].long()
        k, v = (torch.cat([x[pp].view(-1, KV, D)[:P].float().expand(B, P, KV, D), y], 1)
                for x, y in ((s["k"], k), (s["v"], v)))
    w = torch.einsum("bikgd,bjkd->bkgij", q, k).mul_(D ** -0.5)
    j = torch.arange(P + Lk, device="cuda")
    p = P + (s["kv_len"] - q_len)[:, None] + i  # [B, Lq]
    if c["softcap"]:
        w = w.div_(c["softcap"]).tanh_().mul_(c["softcap"])
    if s["slopes"] is not None:
        w -= s["slopes"].view(1, KV, G, 1, 1) * (p[:, :, None] - j).abs()[:, None, None]
    n = (P + s["kv_len"])[:, None]
    hi = n.expand(B, Lq)
    if c["causal"]:
        hi = torch.minimum(hi, p + 1 if s["visible"] is None else torch.maximum(p + 1, s["visible"][:, None]))
    seen = j < hi[:, :, None]
    if c["window"]:
        seen &= j > p[:, :, None] - c["window"]
    w.masked_fill_(~seen[:, None, None], -math.inf)
    top = w.amax(-1, keepdim=True)
    w = w.sub_(top.clamp(min=-3e38)).exp_()
    total = w.sum(-1, keepdim=True)
    o = torch.einsum("bkgij,bjkd->bikgd", w, v) / total.clamp(min=1e-30).permute(0, 3, 1, 2, 4)
    lse = (top + total.log()).permute(0, 3, 1, 2, 4)
    real = i < q_len[:, None]
    out = o.reshape(B, Lq, H, D)[real]
    if s["gate"] is not None:
        out = out / (1 + torch.exp(-s["gate"].float()))
    out = out.to(torch.bfloat16)
    return {"out": out, "lse": lse.reshape(B, Lq, H)[real]} if c["lse"] else {"out": out}


def run(state):
    if own:
        return _run_own(state)
    return {"norm": _run_norm, "append": _run_append, "attention": _run_attention}[state["c"]["kind"]](state)


def exact(case, seed):
    """The definitions in 64 bits, sequence by sequence and head by head."""
    global own
    c, keep = case, own
    own = False
    s = prepare(case, seed)
    own = keep
    if c["kind"] == "norm":
        def rms(t, w):
            return t / (t.square().mean(1, keepdim=True) + 1e-6).sqrt() * (w.double() + c["offset"])
        t = s["x"].double()
        t = t if s["post_w"] is None else rms(t, s["post_w"])
        t = t if s["gate"] is None else t * torch.sigmoid(s["gate"].double())
        r = s["residual"].double() + c["scale"] * t
        return {"residual": r, "y": rms(r, s["pre"])}
    q_len, kv_len = _lengths(c)
    H, KV, D, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    start = np.concatenate([[0], np.cumsum(q_len)])
    if c["kind"] == "append":
        x = s["qkv"].double()
        for w, lo, hi in ((s["qw"], 0, H), (s["kw"], H, H + KV)):
            if w is not None:
                y = x[:, lo:hi]
                x[:, lo:hi] = y / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        half = c["rotary"] // 2
        for f in range(half):
            a = s["pos"][int(s["axis"][f])].double() * s["inv_freq"][f].double()
            e, o = (2 * f, 2 * f + 1) if c["interleaved"] else (f, f + half)
            z = torch.polar(torch.ones_like(a), a)[:, None] * torch.complex(x[:, :H + KV, e], x[:, :H + KV, o])
            x[:, :H + KV, e], x[:, :H + KV, o] = z.real, z.imag
        k, v = s["k"].double(), s["v"].double()
        for b in range(c["seqs"]):
            at = torch.arange(kv_len[b] - q_len[b], kv_len[b], device="cuda")
            t, slot = slice(start[b], start[b + 1]), (s["table"][b, at // page].long(), at % page)
            k[slot], v[slot] = x[t, H:H + KV], x[t, H + KV:]
        return {"q": x[:, :H].contiguous(), "k": k, "v": v}
    G, P = H // KV, c["prefix"]
    out = torch.zeros(s["T"], H, D, dtype=torch.float64, device="cuda")
    lse = torch.full((s["T"], H), -math.inf, dtype=torch.float64, device="cuda")
    for b, (lo, hi) in enumerate(_intervals(c)):
        n, t = kv_len[b], slice(start[b], start[b + 1])
        kk, vv = (torch.cat([x[s["prefix_pages"].long()].reshape(-1, KV, D)[:P],
                             x[s["table"][b].long()].reshape(-1, KV, D)[:n]]) for x in (s["k"], s["v"]))
        j = torch.arange(P + n, device="cuda")
        lo, hi = torch.from_numpy(lo).cuda()[:, None], torch.from_numpy(hi).cuda()[:, None]
        far = (P + n - q_len[b] + torch.arange(q_len[b], device="cuda")[:, None] - j).abs().double()
        for h in range(H):
            z = s["q"][t, h].double() @ kk[:, h // G].double().t() / math.sqrt(D)
            if c["softcap"]:
                z = c["softcap"] * torch.tanh(z / c["softcap"])
            if s["slopes"] is not None:
                z = z - s["slopes"][h].double() * far
            z = torch.where((j >= lo) & (j < hi), z, -math.inf)
            lse[t, h] = torch.logsumexp(z, 1)
            out[t, h] = torch.nan_to_num(torch.softmax(z, 1)) @ vv[:, h // G].double()
    if s["gate"] is not None:
        out = out * torch.sigmoid(s["gate"].double())
    return {"out": out, "lse": lse} if c["lse"] else {"out": out}
