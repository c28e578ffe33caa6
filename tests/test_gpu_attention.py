"""kv_append, paged_attention and norm_residual on the GPU against their
formulas in 64 bits (attention_ref.py), at the sizes and masks where they can
go wrong, and run together as a layer uses them."""
import math

import pytest
import torch

import attention_ref as ref

pytestmark = pytest.mark.gpu


def make(seed, lens, qlens, KV=2, D=128, H=8, page=16, prefix=0, layout="nhd", spare=3, qscale=2.0,
         poison=True, width=None):
    """A shuffled cache with NaN wherever no key was appended."""
    import nvfp4

    g = torch.Generator().manual_seed(seed)
    pages = [-(-n // page) for n in lens]
    pp = -(-prefix // page)
    total = sum(pages) + pp + spare
    order = torch.randperm(total, generator=g).to(torch.int32)
    width = max(max(pages), 1) if width is None else width
    table = torch.full((len(lens), width), -7, dtype=torch.int32)
    at = pp
    for b, p in enumerate(pages):
        table[b, :p] = order[at:at + p]
        at += p
    shape = (total, page, KV, D)
    k, v = (torch.randn(shape, generator=g).to(torch.bfloat16) for _ in range(2))
    if poison:
        used = torch.zeros(total, page, dtype=torch.bool)
        for b, n in enumerate(lens):
            for j in range(n):
                used[table[b, j // page], j % page] = True
        for j in range(prefix):
            used[order[j // page], j % page] = True
        k[~used] = math.nan
        v[~used] = math.nan
    T = sum(qlens)
    q = (qscale * torch.randn(T, H, D, generator=g)).to(torch.bfloat16)
    starts = [0]
    for n in qlens:
        starts.append(starts[-1] + n)
    if layout == "nhd":
        kd, vd = k.cuda(), v.cuda()
    elif layout == "hnd":
        kd, vd = (x.transpose(1, 2).contiguous().cuda().transpose(1, 2) for x in (k, v))
    else:  # one buffer [pages, 2, slot, head, D + 8]
        buf = torch.zeros(total, 2, page, KV, D + 8, dtype=torch.bfloat16)
        buf[:, 0, ..., :D], buf[:, 1, ..., :D] = k, v
        buf = buf.cuda()
        kd, vd = buf[:, 0, ..., :D], buf[:, 1, ..., :D]
    cache = nvfp4.PagedKVCache(kd, vd)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)
    return dict(k=k, v=v, q=q, table=table, kv_len=i32(lens), q_start=i32(starts), cache=cache,
                prefix_pages=order[:pp].clone(), prefix=prefix, T=T, H=H, KV=KV, D=D, g=g)


def batch_of(s, single=None, visible=None, max_q=None):
    import nvfp4

    ql = (s["q_start"][1:] - s["q_start"][:-1])
    single = bool((ql == 1).all()) if single is None else single
    return nvfp4.AttentionBatch(
        s["kv_len"].cuda(), s["table"].cuda(), q_start=None if single else s["q_start"].cuda(),
        num_tokens=s["T"], max_q_len=1 if single else (max_q or int(ql.max())),
        prefix_pages=s["prefix_pages"].cuda() if s["prefix"] else None, prefix_len=s["prefix"],
        visible_len=None if visible is None else visible.cuda())


def run_and_check(s, causal=True, window=0, softcap=0.0, slopes=None, gate=None, visible=None,
                  scale=None, single=None, max_q=None):
    import nvfp4
    from nvfp4 import _lib

    cfg = nvfp4.AttentionConfig(s["H"], s["KV"], s["D"], scale=scale, causal=causal, window=window,
                                softcap=softcap)
    out, lse = nvfp4.paged_attention(
        s["q"].cuda(), s["cache"], batch_of(s, single, visible, max_q), cfg,
        slopes=None if slopes is None else slopes.cuda(), gate=None if gate is None else gate.cuda(),
        return_lse=True)
    torch.cuda.synchronize()
    assert _lib.load().nvfp4_device_status() == 0
    o, l, o_tol, l_tol = ref.attention(
        s["q"], s["k"], s["v"], s["kv_len"], s["table"], s["q_start"],
        prefix_pages=s["prefix_pages"], prefix_len=s["prefix"], visible=visible, scale=scale,
        causal=causal, window=window, softcap=softcap, slopes=slopes, gate=gate)
    ref.check(out, o, o_tol, "out")
    ref.check(lse, l, l_tol, "lse")
    return out, lse


HEADS = [(8, 2, 128), (4, 4, 64), (14, 2, 128), (8, 1, 256), (3, 3, 80), (5, 1, 40), (16, 2, 136)]


@pytest.mark.parametrize("H,KV,D", HEADS)
@pytest.mark.parametrize("page", [16, 64, 256])
def test_single_tokens(H, KV, D, page):
    lens = [1, 15, 16, 17, 63, 64, 65, 130, 1, 257]
    run_and_check(make(1, lens, [1] * len(lens), KV, D, H, page))


def test_one_sequence_split_over_the_gpu():
    """One sequence: its keys go over all blocks and are joined."""
    run_and_check(make(2, [9001], [1], 1, 128, 8, 16))
    run_and_check(make(3, [4097], [1], 2, 256, 16, 64))


@pytest.mark.parametrize("layout", ["hnd", "joint"])
def test_cache_strides(layout):
    run_and_check(make(4, [37, 200, 5], [1, 1, 1], layout=layout))
    run_and_check(make(5, [300, 45], [70, 45], layout=layout))


def test_sequences_without_keys_or_queries():
    """Lengths of zero, a sequence without tokens, more tokens than keys (the
    first of them see nothing)."""
    out, lse = run_and_check(make(6, [0, 3, 0], [1, 1, 1], width=4))
    assert (out[0] == 0).all() and (out[2] == 0).all() and torch.isinf(lse[0]).all()
    run_and_check(make(7, [0, 20, 33], [2, 0, 5], width=4))
    out, lse = run_and_check(make(8, [3, 40], [7, 2], width=4))
    assert (out[:4] == 0).all() and torch.isneginf(lse[:4]).all()


@pytest.mark.parametrize("H,KV,D", HEADS)
@pytest.mark.parametrize("causal", [True, False])
def test_prompts(H, KV, D, causal):
    run_and_check(make(9, [1, 90, 200, 65], [1, 90, 33, 17], KV, D, H, 32), causal=causal)


@pytest.mark.parametrize("H,KV,D", [(8, 1, 128), (8, 1, 256), (2, 2, 64)])
def test_prompts_over_many_key_tiles(H, KV, D):
    """Many key tiles per item and several items per block, repeated: the
    hand-over between the roles of a block, tile after tile."""
    import nvfp4

    s = make(27, [2900, 700, 1500], [300, 700, 40], KV, D, H, 16)
    first, _ = run_and_check(s)
    cfg, b, q = nvfp4.AttentionConfig(H, KV, D), batch_of(s), s["q"].cuda()
    for _ in range(20):
        assert torch.equal(nvfp4.paged_attention(q, s["cache"], b, cfg), first)


@pytest.mark.parametrize("qlens", [[2, 3, 1], [4, 4, 4], [1, 9, 40], [129, 1, 128], [1, 1, 300]])
def test_query_lengths(qlens):
    """Around every row count at which another kernel or tile is taken."""
    lens = [q + 61 * i for i, q in enumerate(qlens)]
    run_and_check(make(10, lens, qlens, 2, 128, 16, 16))
    run_and_check(make(11, lens, qlens, 1, 256, 8, 16))
    run_and_check(make(12, lens, qlens, 4, 64, 4, 64))


@pytest.mark.parametrize("qlens", [[1, 1, 1], [1, 5, 130]])
@pytest.mark.parametrize("opts", [dict(window=1), dict(window=20), dict(window=64), dict(softcap=5.0),
                                  dict(slopes=True), dict(softcap=30.0, slopes=True, window=70),
                                  dict(causal=False, window=33), dict(visible=True),
                                  dict(visible=True, window=50), dict(gate=True), dict(scale=0.3)])
def test_scores_and_masks(qlens, opts):
    o = dict(opts)
    s = make(13, [q + x for q, x in zip(qlens, (0, 150, 77))], qlens, 2, 128, 8, 16)
    if o.pop("slopes", None):
        o["slopes"] = 2.0 ** -torch.arange(1, 9, dtype=torch.float32)
    if o.pop("visible", None):
        o["visible"] = torch.tensor([0, 151, 40], dtype=torch.int32)
    if o.pop("gate", None):
        o["gate"] = torch.randn(s["T"], 8, 128, generator=s["g"]).to(torch.bfloat16)
    run_and_check(s, **o)


@pytest.mark.parametrize("D,H,KV", [(128, 8, 2), (256, 4, 1), (64, 4, 4)])
def test_masks_at_other_head_sizes(D, H, KV):
    qlens = [3, 1, 70]
    s = make(14, [20, 300, 100], qlens, KV, D, H, 32)
    run_and_check(s, window=37, softcap=20.0, slopes=2.0 ** -torch.arange(1, H + 1, dtype=torch.float32),
                  visible=torch.tensor([9, 0, 55], dtype=torch.int32),
                  gate=torch.randn(s["T"], H, D, generator=s["g"]).to(torch.bfloat16))


@pytest.mark.parametrize("prefix", [1, 64, 75, 700])
@pytest.mark.parametrize("qlens", [[1, 1, 1, 1, 1], [1, 20, 3], [1], [200]])
def test_shared_prefix(prefix, qlens):
    lens = [q + 13 * i for i, q in enumerate(qlens)]
    run_and_check(make(15, lens, qlens, 2, 128, 8, 16, prefix=prefix))
    run_and_check(make(16, lens, qlens, 1, 256, 8, 64, prefix=prefix), window=60, softcap=9.0,
                  slopes=2.0 ** -torch.arange(1, 9, dtype=torch.float32))


def test_shared_prefix_is_the_whole_sequence():
    """The same keys as prefix and own part, or all as own: the same result
    within the bound (checked against one reference each), and a query with
    no key of its own sees the prefix."""
    run_and_check(make(17, [0, 5], [0, 1], prefix=33, width=2))
    s = make(18, [0, 2], [1, 1], prefix=40, width=2)
    # kv_len 0 with one query: it stands before the prefix's end.
    run_and_check(s)


@pytest.mark.parametrize("qlens", [[1, 1, 1], [3, 60, 200]])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("prefix", [0, 50])
def test_queries_that_are_not_finite(qlens, gated, prefix):
    """A query with a NaN or an infinity spoils its own row and no other, with
    and without a gate or a prefix part in the last step."""
    import nvfp4

    for D, H, KV in ((128, 8, 2), (256, 8, 1)):
        s = make(28, [q + 70 for q in qlens], qlens, KV, D, H, 16, prefix=prefix)
        gate = torch.randn(s["T"], H, D, generator=s["g"]).to(torch.bfloat16) if gated else None
        bad = s["q"].clone()
        bad[1, 2, 5], bad[s["T"] - 1, 0, 0], bad[0, 4, 1] = math.nan, math.inf, -math.inf
        out = nvfp4.paged_attention(bad.cuda(), s["cache"], batch_of(s), nvfp4.AttentionConfig(H, KV, D),
                                    gate=None if gate is None else gate.cuda())
        hit = [(1, 2), (s["T"] - 1, 0), (0, 4)]
        for t, h in hit:
            assert torch.isnan(out[t, h]).all()
            out[t, h] = 0
        o, _, tol, _ = ref.attention(s["q"], s["k"], s["v"], s["kv_len"], s["table"], s["q_start"],
                                     prefix_pages=s["prefix_pages"], prefix_len=prefix, gate=gate)
        for t, h in hit:
            o[t, h] = 0
        ref.check(out, o, tol, "out")


def test_repeats_bit_for_bit():
    import nvfp4

    s = make(19, [1000, 3, 517, 64], [1, 1, 1, 1], 2, 128, 16, 16)
    cfg = nvfp4.AttentionConfig(16, 2, 128)
    b, q = batch_of(s), s["q"].cuda()
    first = nvfp4.paged_attention(q, s["cache"], b, cfg)
    for _ in range(10):
        assert torch.equal(nvfp4.paged_attention(q, s["cache"], b, cfg), first)


def test_bad_pages_and_lengths_are_clamped():
    """A page id outside the cache reads as zeros; a length beyond the table
    is held to it; a token range beyond the call's rows is cut."""
    s = make(20, [50, 40], [1, 1], 2, 128, 8, 16, poison=False)
    s["table"][0, 1], s["table"][1, 0] = 10 ** 6, -5
    run_and_check(s)
    s = make(21, [64, 40], [1, 1], 2, 128, 8, 16, poison=False, width=4)
    s["kv_len"][0] = 10 ** 6
    run_and_check(s)


def test_rows_outside_every_sequence_stay():
    import nvfp4

    s = make(22, [30, 50], [2, 3], 2, 128, 8, 16)
    cfg = nvfp4.AttentionConfig(8, 2, 128)
    q = torch.cat([s["q"], torch.full((4, 8, 128), math.nan, dtype=torch.bfloat16)]).cuda()
    b = nvfp4.AttentionBatch(s["kv_len"].cuda(), s["table"].cuda(), q_start=s["q_start"].cuda(),
                             num_tokens=9, max_q_len=3)
    out = torch.full((9, 8, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    nvfp4.paged_attention(q, s["cache"], b, cfg, out=out)
    assert (out[5:] == 7).all()
    o, _, tol, _ = ref.attention(s["q"], s["k"], s["v"], s["kv_len"], s["table"], s["q_start"])
    ref.check(out[:5], o, tol, "out")


def test_strided_rows_and_out_in_place():
    import nvfp4

    s = make(23, [30, 50], [2, 30], 2, 128, 8, 16)
    cfg = nvfp4.AttentionConfig(8, 2, 128)
    wide = torch.zeros(s["T"], 8, 2, 128, dtype=torch.bfloat16, device="cuda")  # query and gate side by side
    gate = torch.randn(s["T"], 8, 128, generator=s["g"]).to(torch.bfloat16)
    wide[:, :, 0], wide[:, :, 1] = s["q"].cuda(), gate.cuda()
    q = wide[:, :, 0]
    out = nvfp4.paged_attention(q, s["cache"], batch_of(s), cfg, gate=wide[:, :, 1], out=q)
    assert out.data_ptr() == q.data_ptr()
    o, _, tol, _ = ref.attention(s["q"], s["k"], s["v"], s["kv_len"], s["table"], s["q_start"], gate=gate)
    ref.check(q, o, tol, "out")
    assert torch.equal(wide[:, :, 1].cpu(), gate)


def test_captured_steps_follow_the_device_lengths():
    """One graph, replayed with longer lengths, other queries; two graphs that
    share a workspace, replayed in turn."""
    import nvfp4

    s = make(24, [100, 90, 300], [1, 1, 1], 2, 128, 8, 16)
    t = make(25, [40, 2, 7], [1, 1, 1], 2, 128, 8, 16)
    cfg = nvfp4.AttentionConfig(8, 2, 128)
    graphs = []
    bs, bt = batch_of(s), batch_of(t)
    ws = nvfp4.attention_workspace(cfg, bs)
    for x, b in ((s, bs), (t, bt)):
        q = x["q"].cuda()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            nvfp4.paged_attention(q, x["cache"], b, cfg, workspace=ws)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = nvfp4.paged_attention(q, x["cache"], b, cfg, workspace=ws)
        graphs.append((g, q, out))
    for n in ([100, 90, 300], [17, 90, 299], [64, 1, 128]):
        for x, b, (g, q, out) in ((s, bs, graphs[0]), (t, bt, graphs[1])):
            lens = torch.minimum(torch.tensor(n, dtype=torch.int32), x["kv_len"])
            b.tensors[0].copy_(lens)
            g.replay()
            torch.cuda.synchronize()
            o, _, tol, _ = ref.attention(x["q"], x["k"], x["v"], lens, x["table"], x["q_start"])
            ref.check(out, o, tol, "out")


def test_calls_on_another_stream():
    import nvfp4

    s = make(26, [200, 33], [1, 40], 2, 128, 8, 16)
    cfg = nvfp4.AttentionConfig(8, 2, 128)
    b, q = batch_of(s), s["q"].cuda()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for st in (side, side.cuda_stream):
        out = nvfp4.paged_attention(q, s["cache"], b, cfg, stream=st)
        side.synchronize()
        o, _, tol, _ = ref.attention(s["q"], s["k"], s["v"], s["kv_len"], s["table"], s["q_start"])
        ref.check(out, o, tol, "out")


# ---------------------------------------------------------------- kv_append
def append_case(seed, qlens, ctx, H, KV, D, page, rotary, axes, inter, norm, dtype, far=0, scale=1.0,
                strided=True, offset=0.0):
    import nvfp4

    lens = [a + b for a, b in zip(qlens, ctx)]
    s = make(seed, lens, qlens, KV, D, H, page, poison=False)
    g, T = s["g"], s["T"]
    x = torch.randn(T, H + 2 * KV, D, generator=g).to(dtype)
    dev = x.cuda()
    q, k, v = dev.split([H, KV, KV], 1)
    if not strided:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    inv = axis = pos = rot = None
    if rotary:
        half = rotary // 2
        inv = (1e6 ** (-torch.arange(half, dtype=torch.float64) / half)).float()
        axis = (torch.arange(half) % axes).to(torch.int32) if axes > 1 else None
        rot = nvfp4.Rotary(inv.cuda(), axes=None if axis is None else axis.cuda(), interleaved=inter,
                           scale=scale)
        if axes > 1 or far:
            pos = torch.randint(0, 1000, (axes, T), generator=g, dtype=torch.int32) + far
    w = [(1 - offset + 0.3 * torch.randn(D, generator=g)).to(torch.bfloat16) for _ in range(2)] if norm else [None] * 2
    cu = lambda t: None if t is None else t.cuda()
    before_k, before_v = s["cache"].k.clone(), s["cache"].v.clone()
    got = nvfp4.kv_append(q, k, v, s["cache"], batch_of(s), rotary=rot, positions=cu(pos), q_norm=cu(w[0]),
                          k_norm=cu(w[1]), norm_offset=offset)
    torch.cuda.synchronize()
    X = x.double()
    rq, rk, rv = X.split([H, KV, KV], 1)
    if norm:
        rq, rk = ref.head_norm(rq, w[0], 1e-6, offset), ref.head_norm(rk, w[1], 1e-6, offset)
    own = torch.cat([torch.arange(n - m, n) for n, m in zip(lens, qlens)])
    size = [rq.abs().amax(-1, keepdim=True), rk.abs().amax(-1, keepdim=True)]
    if rotary:
        p = own[None].expand(axes, T) if pos is None else pos
        a = (p[axis.long()] if axis is not None else p[:1].expand(half, T)).double() * inv.double()[:, None]
        rq, rk = ref.rotate(rq, a.T, inter, scale), ref.rotate(rk, a.T, inter, scale)
    # One rounding to bf16, fp32 arithmetic before it: the norm's sum (D + 8
    # roundings at most, halved by the root), the angle (2^-23 turns = 2^-20)
    # and sincos (2 units) on values of the row's size.
    tol = lambda r, z: ref.BF16 * r.abs() + (1 + ref.BF16) * z * max(scale, 1) * (ref.F32 * (D + 40) + 2.0 ** -20)
    ref.check(got, rq, tol(rq, size[0]), "q")
    want_k, want_v = before_k.double().cpu(), before_v.double().cpu()
    tk, tv = torch.zeros_like(want_k), torch.zeros_like(want_v)
    seq = torch.repeat_interleave(torch.arange(len(qlens)), torch.tensor(qlens))
    at = (s["table"][seq, own // page].long(), own % page)
    want_k[at], want_v[at] = rk, rv
    tk[at], tv[at] = tol(rk, size[1]), ref.BF16 * rv.abs()
    ref.check(s["cache"].k, want_k, tk, "k")
    ref.check(s["cache"].v, want_v, tv, "v")


@pytest.mark.parametrize("H,KV,D", HEADS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("qlens,ctx", [([1] * 5, [0, 15, 16, 40, 3]), ([1, 17, 0, 40], [0, 3, 9, 30])])
def test_append(H, KV, D, dtype, qlens, ctx):
    append_case(30, qlens, ctx, H, KV, D, 16, D if D % 16 == 0 else D // 2, 1, False, True, dtype)


@pytest.mark.parametrize("rotary", [0, 2, 6, 16, 64, 126, 128])
@pytest.mark.parametrize("axes,inter", [(1, False), (1, True), (3, False), (3, True)])
def test_append_rotations(rotary, axes, inter):
    append_case(31, [3, 1, 8], [5, 0, 100], 4, 2, 128, 32, rotary, axes, inter, rotary % 4 == 0, torch.bfloat16)


def test_append_far_positions_scale_and_offset():
    append_case(32, [5, 2], [0, 0], 4, 2, 128, 16, 128, 1, False, True, torch.float32, far=1_000_000)
    append_case(33, [5, 2], [0, 0], 4, 2, 64, 16, 64, 3, False, True, torch.float32, far=2_000_000_000)
    append_case(34, [5, 2], [0, 9], 4, 2, 256, 16, 64, 3, True, True, torch.bfloat16, scale=1.3, offset=1.0,
                strided=False)


def test_append_many_tokens():
    append_case(35, [900, 1, 700], [0, 5, 64], 8, 2, 128, 16, 128, 1, False, True, torch.bfloat16)


def test_append_skips_what_has_no_place():
    """Keys before the first position or beyond the table, bad pages, rows in
    no sequence: nothing else changes."""
    import nvfp4

    s = make(36, [2, 32], [4, 3], 2, 128, 4, 16, poison=False, width=2)
    s["table"][1, 0] = -1
    s["kv_len"] = torch.tensor([2, 34], dtype=torch.int32)  # b = 1: keys 31 .. 33, page 2 missing
    x = torch.randn(9, 8, 128, generator=s["g"]).to(torch.bfloat16).cuda()
    q, k, v = x.split([4, 2, 2], 1)
    b = nvfp4.AttentionBatch(s["kv_len"].cuda(), s["table"].cuda(), q_start=s["q_start"].cuda(),
                             num_tokens=9, max_q_len=4)
    k0, v0 = s["cache"].k.clone(), s["cache"].v.clone()
    out = torch.full((9, 4, 128), 5.0, dtype=torch.bfloat16, device="cuda")
    nvfp4.kv_append(q, k, v, s["cache"], b, q_out=out)
    assert torch.equal(out[:7], q[:7]) and (out[7:] == 5).all()
    for c, c0, x in ((s["cache"].k, k0, k), (s["cache"].v, v0, v)):
        want = c0.clone()
        want[s["table"][0, 0], 0:2] = x[2:4]
        want[s["table"][1, 1], 15] = x[4]
        assert torch.equal(c, want)


def test_append_in_place_keeps_the_rest():
    import nvfp4

    s = make(37, [9, 5], [2, 5], 2, 128, 4, 16, poison=False)
    x = torch.randn(7, 8, 128, generator=s["g"]).to(torch.bfloat16).cuda()
    q, k, v = x.split([4, 2, 2], 1)
    inv = torch.rand(64, generator=s["g"]).cuda()
    want = nvfp4.kv_append(q, k, v, s["cache"], batch_of(s), rotary=nvfp4.Rotary(inv))
    kv = x[:, 4:].clone()
    got = nvfp4.kv_append(q, k, v, s["cache"], batch_of(s), rotary=nvfp4.Rotary(inv), q_out=q)
    assert torch.equal(got, want) and torch.equal(x[:, 4:], kv)


# ------------------------------------------------------------ norm_residual
@pytest.mark.parametrize("rows,hidden", [(1, 1), (3, 7), (1, 2048), (5, 64), (33, 100), (2, 4096), (4, 5120),
                                         (2, 8200), (2, 16384), (1, 32768), (300, 256), (1, 9999)])
@pytest.mark.parametrize("x_dtype,r_dtype", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                             (torch.float32, torch.float32)])
@pytest.mark.parametrize("post,gate,act", [(False, None, "sigmoid"), (True, "full", "sigmoid"),
                                           (True, "token", "linear"), (False, "channel", "sigmoid")])
def test_norm_residual(rows, hidden, x_dtype, r_dtype, post, gate, act):
    import nvfp4

    g = torch.Generator().manual_seed(rows * 100003 + hidden)
    n = lambda *s: torch.randn(*s, generator=g)
    x, r = n(rows, hidden).to(x_dtype), (3 * n(rows, hidden)).to(r_dtype)
    wp, wq = ((1 + 0.2 * n(hidden)).to(torch.bfloat16) for _ in range(2))
    gt = None if gate is None else n(*{"full": (rows, hidden), "token": (rows, 1), "channel": (hidden,)}[gate]).to(torch.bfloat16)
    cu = lambda t: None if t is None else t.cuda()
    ro, y = nvfp4.norm_residual(x.cuda(), r.cuda(), pre_weight=wq.cuda(), post_weight=wp.cuda() if post else None,
                                gate=cu(gt), gate_act=act, scale=0.75, weight_offset=0.5)
    u = x.double()
    if post:
        u = ref.head_norm(u, wp, 1e-6, 0.5)
    if gt is not None:
        u = u * (torch.sigmoid(gt.double()) if act == "sigmoid" else gt.double())
    R = r.double() + 0.75 * u
    Y = ref.head_norm(R, wq, 1e-6, 0.5)
    # fp32: the sum of squares (up to 32 terms per thread and 10 halvings, its
    # error halved by the root), the gate and a handful of products.
    rel = 48 * ref.F32
    step = lambda t, dt: t.abs() * (ref.BF16 if dt == torch.bfloat16 else ref.F32)
    err = rel * (0.75 * u.abs() + R.abs())
    ref.check(ro, R, err + step(R, r_dtype), "residual")
    spread = err / R.square().mean(-1, keepdim=True).add(1e-6).sqrt() * (wq.double() + 0.5).abs()
    ref.check(y, Y, spread + rel * Y.abs() + step(Y, torch.bfloat16) * 1.01, "y")


def test_norm_forms():
    """Parts left out, strided rows, updates in place, fp32 output."""
    import nvfp4

    g = torch.Generator().manual_seed(5)
    wide = torch.randn(6, 3, 128, generator=g).to(torch.bfloat16).cuda()
    w = (1 + 0.2 * torch.randn(128, generator=g)).to(torch.bfloat16).cuda()
    x = wide[:, 1]
    r, y = nvfp4.norm_residual(x, pre_weight=w, y_dtype=torch.float32)
    assert torch.equal(r, x)
    Y = ref.head_norm(x.double().cpu(), w.cpu(), 1e-6, 0.0)
    ref.check(y, Y, 48 * ref.F32 * Y.abs(), "y")
    r2, none = nvfp4.norm_residual(x, wide[:, 0])
    assert none is None and torch.equal(r2, (x.float() + wide[:, 0].float()).to(torch.bfloat16))
    other = wide[:, 2].clone()
    res = wide[:, 0].clone()
    a, b = nvfp4.norm_residual(x, wide[:, 0], pre_weight=w, residual_out=wide[:, 0])
    assert a.data_ptr() == wide.data_ptr() and torch.equal(wide[:, 0], r2) and torch.equal(wide[:, 2], other)
    c, d = nvfp4.norm_residual(x.contiguous(), res, pre_weight=w)
    assert torch.equal(a, c) and torch.equal(b, d)
    odd = torch.randn(5, 131, generator=g).to(torch.bfloat16).cuda()[:, 1:129]  # rows off 16 bytes
    _, y = nvfp4.norm_residual(odd, pre_weight=w)
    _, z = nvfp4.norm_residual(odd.contiguous(), pre_weight=w)
    assert torch.equal(y, z) or (y.float() - z.float()).abs().max() <= 2 * ref.BF16 * z.float().abs().max()
    empty = nvfp4.norm_residual(x[:0], pre_weight=w)
    assert empty[1].shape == (0, 128)


def test_rows_of_zeros_and_not_finite():
    import nvfp4

    x = torch.zeros(3, 256, dtype=torch.bfloat16, device="cuda")
    x[1, 3], x[2, 0] = math.inf, math.nan
    w = torch.ones(256, dtype=torch.bfloat16, device="cuda")
    _, y = nvfp4.norm_residual(x, pre_weight=w)
    assert (y[0] == 0).all() and torch.isnan(y[1, 3]) and (y[1, 4:] == 0).all() and torch.isnan(y[2]).all()
