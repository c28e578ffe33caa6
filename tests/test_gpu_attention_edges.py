"""What paged_attention, kv_append, norm_residual and AttentionLayer must also
get right: large caps, distances beyond 2^24, values that are not finite, rows
in no sequence, loops beyond their first turn."""
import math

import pytest
import torch

import attention_ref as ref
from test_gpu_attention import append_case, batch_of, make, run_and_check, test_norm_residual as norm_case

pytestmark = pytest.mark.gpu
I32_MAX = 2 ** 31 - 1


@pytest.mark.parametrize("qlens", [[1, 1, 1, 1], [2, 40, 1, 9]])
def test_one_page_table_row_for_all_sequences(qlens):
    """Parallel samples over the same pages: one row, expanded, against a row each."""
    import nvfp4

    H, KV, D, page, pages = 8, 2, 128, 16, 6
    g = torch.Generator().manual_seed(89)
    row = torch.tensor([[3, 0, 5, 1, 4, 2]], dtype=torch.int32, device="cuda")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    # Each sequence appends to keys of its own, behind the ones before.
    ends = torch.tensor(qlens).cumsum(0).tolist()
    x = torch.randn(sum(qlens), H + 2 * KV, D, generator=g).to(torch.bfloat16).cuda()
    q, k, v = x.split([H, KV, KV], 1)
    got = []
    for table in (row.expand(4, -1), row.repeat(4, 1)):
        cache = nvfp4.PagedKVCache(*(torch.full((pages, page, KV, D), 0.5, dtype=torch.bfloat16, device="cuda")
                                     for _ in range(2)))
        batch = nvfp4.AttentionBatch(i32([n + 20 for n in ends]), table, q_start=i32([0] + ends),
                                     num_tokens=sum(qlens), max_q_len=max(qlens))
        turned = nvfp4.kv_append(q, k, v, cache, batch)
        got.append((turned, cache.k, cache.v, nvfp4.paged_attention(turned, cache, batch,
                                                                    nvfp4.AttentionConfig(H, KV, D))))
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert not (got[0][1] == 0.5).all()


@pytest.mark.parametrize("H,KV,D", [(8, 2, 128), (8, 1, 256), (4, 4, 64)])
@pytest.mark.parametrize("prefix", [0, 70])
def test_out_over_the_gate(H, KV, D, prefix):
    """Each value of the gate is read before the output takes its place: in the
    item's own end, in the join of cut items and behind a prefix."""
    import nvfp4

    for lens, qlens in (([9000, 3, 40], [1, 1, 1]), ([3000, 300, 70], [260, 300, 1])):
        s = make(87, lens, qlens, KV, D, H, 16, prefix=prefix)
        gate = torch.randn(s["T"], H, D, generator=s["g"]).to(torch.bfloat16).cuda()
        cfg, b, q = nvfp4.AttentionConfig(H, KV, D), batch_of(s), s["q"].cuda()
        want = nvfp4.paged_attention(q, s["cache"], b, cfg, gate=gate)
        got = nvfp4.paged_attention(q, s["cache"], b, cfg, gate=gate, out=gate)
        assert got.data_ptr() == gate.data_ptr() and torch.equal(got, want)
        in_place = nvfp4.paged_attention(q, s["cache"], b, cfg, gate=want.clone(), out=q)
        assert in_place.data_ptr() == q.data_ptr() and torch.isfinite(in_place).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rotary,inter", [(0, False), (64, False), (64, True), (6, False), (128, False)])
@pytest.mark.parametrize("norm", [False, True])
def test_append_of_values_that_are_not_finite(dtype, rotary, inter, norm):
    """What is not turned passes by itself: an infinity or a NaN stays in its
    place, and in its pair where that is turned."""
    import nvfp4

    H, KV, D, qlens = 4, 2, 128, [3, 5]
    s = make(90, [n + 9 for n in qlens], qlens, KV, D, H, 16, poison=False)
    T = s["T"]
    x = torch.randn(T, H + 2 * KV, D, generator=s["g"]).to(dtype)
    x[0, 0, 3], x[1, 1, 70], x[2, 2, 127], x[3, 3, 100] = math.inf, -math.inf, math.nan, math.inf
    x[4, H, 65], x[5, H + 1, 126], x[6, H + KV, 9], x[7, H + KV + 1, 64] = -math.inf, math.nan, math.inf, -math.inf
    inv = (1e4 ** (-torch.arange(rotary // 2, dtype=torch.float64) / max(rotary // 2, 1))).float()
    w = (1 + 0.3 * torch.randn(D, generator=s["g"])).to(torch.bfloat16) if norm else None
    cu = lambda t: None if t is None else t.cuda()
    q, k, v = x.cuda().split([H, KV, KV], 1)
    got = nvfp4.kv_append(q, k, v, s["cache"], batch_of(s), q_norm=cu(w), k_norm=cu(w),
                          rotary=nvfp4.Rotary(inv.cuda(), interleaved=inter) if rotary else None)
    rows = x.double()
    if norm:
        rows = torch.cat([ref.head_norm(rows[:, :H + KV], w, 1e-6, 0.0), rows[:, H + KV:]], 1)
    own = torch.cat([torch.arange(n - m, n) for n, m in zip(s["kv_len"].tolist(), qlens)])
    if rotary:
        rows = torch.cat([ref.rotate(rows[:, :H + KV], own[:, None].double() * inv.double(), inter),
                          rows[:, H + KV:]], 1)
    seq = torch.repeat_interleave(torch.arange(2), torch.tensor(qlens))
    at = (s["table"][seq, own // 16].long(), own % 16)
    got = torch.cat([got.cpu(), s["cache"].k.cpu()[at], s["cache"].v.cpu()[at]], 1)
    # As for the finite rows: one rounding to bf16 and fp32 before it.
    size = torch.where(torch.isfinite(rows), rows, 0.0).abs().amax(-1, keepdim=True)
    ref.check(got, rows, ref.BF16 * rows.abs() + 1.01 * size * (ref.F32 * (D + 40) + 2.0 ** -20), "rows")


@pytest.mark.parametrize("cap", [0.5, 3.0, 50.0, 1e3, 1e4, 1e6, 1e20, 3e38])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("tokens", [1, 3, 90])
def test_caps_of_every_size(cap, D, tokens):
    """One key per query (window 1), so that the log-sum-exp is the capped
    score itself: its error goes with the score and not with the cap."""
    import nvfp4

    H, KV, qlens = 4, 1, [tokens, tokens, tokens]
    s = make(91, [tokens + 40, tokens, tokens + 3], qlens, KV, D, H, 16)
    _, lse = nvfp4.paged_attention(s["q"].cuda(), s["cache"], batch_of(s),
                                   nvfp4.AttentionConfig(H, KV, D, window=1, softcap=cap), return_lse=True)
    own = torch.cat([torch.arange(n - tokens, n) for n in s["kv_len"].tolist()])
    seq = torch.repeat_interleave(torch.arange(3), tokens)
    key = s["k"][s["table"][seq, own // 16].long(), own % 16, 0].double()
    x = s["q"].double()
    want = torch.einsum("thd,td->th", x, key) / math.sqrt(D)
    size = torch.einsum("thd,td->th", x.abs(), key.abs()) / math.sqrt(D)
    c64 = float(torch.tensor(cap, dtype=torch.float32))
    want = c64 * torch.tanh(want / c64)
    # The product's sum and the scale: D + 4 roundings of its terms' size, which
    # the cap never enlarges; then the cap in fp32 (16 roundings of the result)
    # and the way to base 2 and back (4).
    ref.check(lse, want, ref.F32 * ((D + 4) * size + 20 * want.abs()), "lse")


@pytest.mark.parametrize("qlens", [[1, 1, 1], [3, 60, 200]])
@pytest.mark.parametrize("D,H,KV", [(128, 8, 2), (256, 8, 1), (64, 8, 2)])
def test_capped_scores_that_are_not_finite(qlens, D, H, KV):
    """A cap holds an infinite score and keeps one that is not a number."""
    import nvfp4

    s = make(86, [q + 70 for q in qlens], qlens, KV, D, H, 16)
    bad, big = s["q"].clone(), s["q"].clone()
    bad[1, 2, 5] = math.nan
    # Scores beyond fp32: one column of q and of every key decides their sign.
    big[0, 4] = 0
    big[0, 4, 1] = 3e38
    k = s["cache"].k.clone()
    used = torch.isfinite(k).all(-1)
    k[..., 1] = torch.where(used, torch.where(k[..., 1] > 0, 2.0, -2.0).to(torch.bfloat16), k[..., 1])
    cache = nvfp4.PagedKVCache(k, s["cache"].v)
    cfg = nvfp4.AttentionConfig(H, KV, D, scale=1.0, softcap=4.0)
    b = batch_of(s)
    out = nvfp4.paged_attention(bad.cuda(), s["cache"], b, nvfp4.AttentionConfig(H, KV, D, softcap=4.0))
    assert torch.isnan(out[1, 2]).all()
    out[1, 2] = 0
    assert torch.isfinite(out).all()
    out, lse = nvfp4.paged_attention(big.cuda(), cache, b, cfg, return_lse=True)
    big[0, 4, 1] = 1e6  # far beyond the cap, within fp32: the same capped scores
    want, want_lse = nvfp4.paged_attention(big.cuda(), cache, b, cfg, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, want_lse) and torch.isfinite(lse).all()


@pytest.mark.parametrize("n", [2 ** 24 + 2, 2 ** 25 + 77])
@pytest.mark.parametrize("tokens", [1, 4, 70])
@pytest.mark.parametrize("D", [64, 128])
def test_distances_at_far_positions(n, tokens, D):
    """The bias goes by whole distances, also where fp32 no longer holds the
    positions.  A window keeps the keys few; the table names eight pages in turn."""
    import nvfp4

    H, KV, page, window = 4, 1, 256, 50
    g = torch.Generator().manual_seed(92)
    k, v = (torch.randn(8, page, KV, D, generator=g).to(torch.bfloat16) for _ in range(2))
    q = torch.randn(tokens, H, D, generator=g).to(torch.bfloat16)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    table = (torch.arange(-(-n // page), device="cuda") % 8).to(torch.int32)[None]
    batch = nvfp4.AttentionBatch(i32([n]), table, q_start=i32([0, tokens]), num_tokens=tokens, max_q_len=tokens)
    slopes = torch.tensor([1.0, 0.5, 0.25, 2.0])
    out, lse = nvfp4.paged_attention(q.cuda(), nvfp4.PagedKVCache(k.cuda(), v.cuda()), batch,
                                     nvfp4.AttentionConfig(H, KV, D, window=window), slopes=slopes.cuda(),
                                     return_lse=True)
    # The same as a short sequence: the last keys alone, behind a multiple of the eight pages.
    first = (n - tokens - window) // (8 * page) * (8 * page)
    o, l, o_tol, l_tol = ref.attention(q, k, v, [n - first], (torch.arange(-(-(n - first) // page)) % 8)[None],
                                       [0, tokens], window=window, slopes=slopes)
    ref.check(out, o, o_tol, "out")
    ref.check(lse, l, l_tol, "lse")


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [I32_MAX, I32_MAX - 3, 2 ** 30, 2 ** 30 + 1])
def test_windows_as_long_as_the_type(causal, window):
    """A window beyond every sequence masks nothing, also for the tokens that
    stand before the first key."""
    run_and_check(make(8, [3, 40], [7, 2], width=4), causal=causal, window=window)
    run_and_check(make(93, [30, 9], [200, 9], 1, 128, 8, 16), causal=causal, window=window)
    run_and_check(make(94, [3, 0, 40], [70, 1, 2], 2, 64, 8, 16, prefix=20), causal=causal, window=window)


@pytest.mark.parametrize("last", [8, 9, I32_MAX])
def test_append_holds_token_ranges_to_the_calls_rows(last):
    """Tokens beyond the call's rows do not exist: those that do are the last
    ones of their sequence's keys, for the append as for the attention."""
    import nvfp4

    s = make(95, [12, 20], [3, 4], 2, 128, 4, 16, poison=False)
    x = torch.randn(7, 8, 128, generator=s["g"]).to(torch.bfloat16).cuda()
    q, k, v = x.split([4, 2, 2], 1)
    starts = s["q_start"].clone()
    starts[2] = last
    b = nvfp4.AttentionBatch(s["kv_len"].cuda(), s["table"].cuda(), q_start=starts.cuda(), num_tokens=7, max_q_len=4)
    want = [c.clone() for c in (s["cache"].k, s["cache"].v)]
    for c, rows in zip(want, (k, v)):
        for t, (seq, key) in enumerate([(0, 9), (0, 10), (0, 11), (1, 16), (1, 17), (1, 18), (1, 19)]):
            c[s["table"][seq, key // 16], key % 16] = rows[t]
    got = nvfp4.kv_append(q, k, v, s["cache"], b)
    assert torch.equal(got, q)
    assert torch.equal(s["cache"].k, want[0]) and torch.equal(s["cache"].v, want[1])


def test_one_row_of_positions_for_all_axes():
    """Text under a rotation by time, height and width: [T] expanded to the axes."""
    import nvfp4

    s = make(88, [40, 9], [30, 9], 2, 128, 4, 16, poison=False)
    T = s["T"]
    q, k, v = torch.randn(T, 8, 128, generator=s["g"]).to(torch.bfloat16).cuda().split([4, 2, 2], 1)
    pos = torch.randint(0, 5000, (T,), generator=s["g"], dtype=torch.int32).cuda()
    rot = nvfp4.Rotary(torch.rand(64, generator=s["g"]).cuda(), axes=(torch.arange(64) % 3).to(torch.int32).cuda())
    got = []
    for positions in (pos.expand(3, -1), pos.repeat(3, 1)):
        turned = nvfp4.kv_append(q, k, v, s["cache"], batch_of(s), rotary=rot, positions=positions)
        got.append((turned, s["cache"].k.clone()))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    with pytest.raises(ValueError, match="overlap"):
        nvfp4.kv_append(q, k, v, s["cache"], batch_of(s), rotary=rot,
                        positions=torch.zeros(T + 4, dtype=torch.int32, device="cuda").as_strided((3, T), (2, 1)))


LONG = [([2300, 1, 149], [0, 40, 17]), ([2500], [3])]


@pytest.mark.parametrize("H,KV,D", [(32, 6, 64), (14, 3, 128), (7, 2, 256), (11, 3, 136)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("form", ["halves", "interleaved", "by element", "plain"])
def test_append_of_long_prompts(H, KV, D, dtype, form):
    """A warp takes a whole token: every ring slot is filled more than twice, and
    the heads' kind changes inside the ring."""
    rotary = {"halves": D // 2 if D % 16 == 0 else 64, "interleaved": D, "by element": 12, "plain": 0}[form]
    for i, (qlens, ctx) in enumerate(LONG):
        append_case(96 + i, qlens, ctx, H, KV, D, 32, rotary, 3 if i else 1, form == "interleaved", form != "plain",
                    dtype)


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_of_long_prompts_in_place_and_off_alignment(inter, dtype):
    """q_out over q, and rows that start off 16 bytes, against packed rows."""
    import nvfp4

    H, KV, D, T = 14, 3, 128, 2400
    s = make(98, [T + 5], [T], KV, D, H, 32, poison=False)
    x = torch.randn(T, H + 2 * KV, D, generator=s["g"]).to(dtype).cuda()
    rot = nvfp4.Rotary(torch.rand(32, generator=s["g"]).cuda(), interleaved=inter)
    w = (1 + 0.2 * torch.randn(D, generator=s["g"])).to(torch.bfloat16).cuda()

    def run(x, **kw):
        q, k, v = x.split([H, KV, KV], 1)
        s["cache"].k.zero_(), s["cache"].v.zero_()
        got = nvfp4.kv_append(q, k, v, s["cache"], batch_of(s), rotary=rot, q_norm=w, k_norm=w,
                              **{n: q for n in kw})
        return got.clone(), s["cache"].k.clone(), s["cache"].v.clone()

    want = run(x)
    odd = torch.empty(T, H + 2 * KV, D + 1, dtype=dtype, device="cuda")[..., 1:]
    odd.copy_(x)
    for a, b in zip(run(odd), want):
        # Each within half a step of the exact value, and its fp32 error.
        assert ((a.double() - b.double()).abs() <= 2 * ref.BF16 * b.double().abs() + 2.0 ** -18 * 8).all()
    if dtype is torch.bfloat16:
        for a, b in zip(run(x, q_out=1), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("rows", [591, 592, 2003])
@pytest.mark.parametrize("hidden", [8, 100, 264, 512, 520, 1024, 2048, 5000])
@pytest.mark.parametrize("x_dtype,r_dtype,post,gate,act", [
    (torch.bfloat16, torch.bfloat16, False, None, "sigmoid"), (torch.bfloat16, torch.float32, True, "token", "sigmoid"),
    (torch.float32, torch.float32, True, "full", "linear"), (torch.bfloat16, torch.float32, False, "channel", "sigmoid")])
def test_norm_of_many_rows(rows, hidden, x_dtype, r_dtype, post, gate, act):
    norm_case(rows, hidden, x_dtype, r_dtype, post, gate, act)


@pytest.mark.parametrize("rows,hidden", [(600, 8192), (593, 16384), (593, 9000), (40, 32768)])
def test_norm_of_many_long_rows(rows, hidden):
    norm_case(rows, hidden, torch.bfloat16, torch.float32, True, "full", "sigmoid")


@pytest.mark.parametrize("rows,hidden", [(593, 8), (593, 512), (700, 520), (700, 2048), (600, 8200)])
def test_norm_of_many_rows_off_alignment(rows, hidden):
    import nvfp4

    g = torch.Generator().manual_seed(hidden)
    n = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).cuda()
    w, p, gate = n(hidden), n(hidden), n(rows, 1)
    odd, res = n(rows, hidden + 1)[:, 1:], n(rows, hidden + 3)[:, 3:]
    got = nvfp4.norm_residual(odd, res, pre_weight=w, post_weight=p, gate=gate)
    r, y = nvfp4.norm_residual(odd.contiguous(), res.contiguous(), pre_weight=w, post_weight=p, gate=gate)
    for a, b, scale in ((got[0], r, 1.0), (got[1], y, 1.0)):
        # The sums' order differs: both within half a step and 48 fp32 roundings of the exact value.
        tol = 2 * (ref.BF16 + 48 * ref.F32) * b.double().abs() + 2 * 48 * ref.F32 * b.double().abs().amax(1, keepdim=True)
        assert ((a.double() - b.double()).abs() <= tol).all()
