"""An attention layer end to end: loaded NVFP4 projections, norms, cache,
rotation, attention, gate; a prompt, then single tokens, against the same layer
in 64 bits, and a captured decode step.

Tolerance (max |err| / RMS): 2e-2, that of the library's bf16 paths (two
projections with bf16 operands and results, the attention between them)."""
import math
from types import SimpleNamespace

import pytest
import torch

import attention_ref as ref

pytestmark = pytest.mark.gpu


def loaded(O, rng, out, cols, per_row):
    from nvfp4 import synthetic
    from nvfp4.weight_loader import LoadedWeight

    wd = synthetic.linear_weights(out, cols, seed=int(rng.integers(1 << 30)))
    ins = 0.75
    ws2 = torch.from_numpy(wd["ws2"])
    if not per_row:
        ws2 = torch.full((out,), float(ws2[0]))
    lw = LoadedWeight(torch.from_numpy(wd["w"]).cuda(), torch.from_numpy(wd["sf"]).cuda(), float(ws2[0]), ins, out,
                      cols, ws2.cuda() if per_row else None)
    dense = torch.from_numpy(O.dequant(wd["w"], wd["sf"])).double() * (ws2.double() * ins)[:, None]
    return lw, dense


def build(O, seed, H, KV, D, d_model, gated, rotary):
    import numpy as np
    import nvfp4

    rng = np.random.default_rng(seed)
    g = torch.Generator().manual_seed(seed)
    nq = H * (2 if gated else 1)
    q, dq = loaded(O, rng, nq * D, d_model, True)
    k, dk = loaded(O, rng, KV * D, d_model, False)
    v, dv = loaded(O, rng, KV * D, d_model, True)
    o, do = loaded(O, rng, d_model, H * D, True)
    w = lambda n: (1 + 0.2 * torch.randn(n, generator=g)).to(torch.bfloat16)
    raw = lambda t: t.view(torch.uint8).numpy()
    norms = dict(input=w(d_model), post=w(d_model), q=w(D), k=w(D))
    layer = SimpleNamespace(q_proj=q, k_proj=k, v_proj=v, o_proj=o, input_layernorm=raw(norms["input"]),
                            post_attn_layernorm=raw(norms["post"]))
    weights = nvfp4.AttentionWeights.from_layer(layer, norms["q"], norms["k"])
    half = rotary // 2
    inv = (1e4 ** (-torch.arange(half, dtype=torch.float64) / half)).float()
    att = nvfp4.AttentionLayer(weights, nvfp4.AttentionConfig(H, KV, D), nvfp4.Rotary(inv.cuda()), gated=gated)
    return att, dict(w=torch.cat([dq, dk, dv]), o=do, inv=inv, gated=gated, H=H, KV=KV, D=D, **norms)


def reference(m, hidden, past):
    """One sequence: hidden [n, d_model] 64 bits, past (k, v) lists; returns
    the residual and normed output."""
    H, KV, D = m["H"], m["KV"], m["D"]
    h = ref.head_norm(hidden, m["input"], 1e-6, 0.0)
    x = h @ m["w"].T
    n = hidden.shape[0]
    nq = H * (2 if m["gated"] else 1)
    heads = x.view(n, nq + 2 * KV, D)
    q, k, v = heads[:, :nq], heads[:, nq:nq + KV], heads[:, nq + KV:]
    gate = None
    if m["gated"]:
        both = q.reshape(n, H, 2, D)
        q, gate = both[:, :, 0], both[:, :, 1]
    at = past[0].shape[0] + torch.arange(n)
    ang = at[:, None].double() * m["inv"].double()[None]
    q = ref.rotate(ref.head_norm(q, m["q"], 1e-6, 0.0), ang, False)
    k = ref.rotate(ref.head_norm(k, m["k"], 1e-6, 0.0), ang, False)
    past[0], past[1] = torch.cat([past[0], k]), torch.cat([past[1], v])
    s = torch.einsum("ihd,jhd->hij", q, past[0].repeat_interleave(H // KV, 1)) / math.sqrt(D)
    s = s.masked_fill(torch.arange(past[0].shape[0])[None, None] > at[None, :, None], -math.inf)
    a = torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), past[1].repeat_interleave(H // KV, 1))
    if gate is not None:
        a = a * torch.sigmoid(gate)
    r = hidden + a.reshape(n, H * D) @ m["o"].T
    return r, ref.head_norm(r, m["post"], 1e-6, 0.0)


def close(got, want):
    err = float((got.double().cpu() - want).abs().max() / want.square().mean().sqrt())
    assert err <= 2e-2, err


@pytest.mark.parametrize("H,KV,D,gated,rotary,res", [(8, 2, 128, False, 128, torch.bfloat16),
                                                     (8, 1, 256, True, 64, torch.float32),
                                                     (4, 4, 64, False, 32, torch.float32)])
def test_prompt_then_tokens(O, H, KV, D, gated, rotary, res):
    import nvfp4

    d_model, page = 512, 16
    att, m = build(O, 7, H, KV, D, d_model, gated, rotary)
    g = torch.Generator().manual_seed(3)
    lens = [37, 80]
    cache = nvfp4.PagedKVCache.empty(16, page, KV, D)
    cache.k.fill_(math.nan)
    cache.v.fill_(math.nan)
    table = torch.randperm(16, generator=g)[:14].view(2, 7).to(torch.int32).cuda()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    past = [[torch.zeros(0, KV, D, dtype=torch.float64) for _ in range(2)] for _ in lens]
    first = torch.randn(sum(lens), d_model, generator=g).to(res)
    batch = nvfp4.AttentionBatch(i32(lens), table, q_start=i32([0, lens[0], sum(lens)]), num_tokens=sum(lens),
                                 max_q_len=max(lens))
    r, y = att.step(None, first.cuda(), cache, batch)
    want = [reference(m, x, p) for x, p in zip(first.double().split(lens), past)]
    close(r, torch.cat([w[0] for w in want]))
    close(y, torch.cat([w[1] for w in want]))

    kv = i32(lens)
    one = nvfp4.AttentionBatch(kv, table)
    ws = nvfp4.attention_workspace(att.config, one)
    x_in = torch.zeros(2, d_model, dtype=torch.bfloat16, device="cuda")
    r_in = torch.zeros(2, d_model, dtype=res, device="cuda")
    graph = None
    for step in range(4):  # the last two replay a captured step
        x = torch.randn(2, d_model, generator=g).to(torch.bfloat16)
        h = torch.randn(2, d_model, generator=g).to(res)
        kv += 1
        x_in.copy_(x)
        r_in.copy_(h)
        if step < 2:
            r, y = att.step(x_in, r_in, cache, one, workspace=ws)
        else:
            if graph is None:
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    r, y = att.step(x_in, r_in, cache, one, workspace=ws)
            graph.replay()
        torch.cuda.synchronize()
        stream_in = (x.double() + h.double()).to(res).double()
        want = [reference(m, stream_in[b:b + 1], past[b]) for b in range(2)]
        close(r, torch.cat([w[0] for w in want]))
        close(y, torch.cat([w[1] for w in want]))
