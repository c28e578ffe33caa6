"""How paged_attention divides a call's work: items cut into few and into many
parts side by side, the ways of planning (few, many and very many sequences,
with few and with many items), bounds that are larger than the lengths, and
two calls at once."""
import pytest
import torch

from test_gpu_attention import batch_of, make, run_and_check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H,KV,D", [(8, 1, 64), (8, 2, 128), (16, 2, 256), (6, 2, 80), (4, 4, 136)])
@pytest.mark.parametrize("tokens", [1, 2])
def test_long_contexts_beside_short_ones(H, KV, D, tokens):
    lens = [20011, 2, 40, 700, 3, 65, 31, 1300, 2]
    run_and_check(make(71, lens, [tokens] * len(lens), KV, D, H, 64))


def test_long_contexts_behind_a_prefix():
    s = make(72, [9000, 2, 300], [1, 1, 1], 1, 256, 8, 16, prefix=5000)
    gate = torch.randn(s["T"], s["H"], s["D"], generator=s["g"]).to(torch.bfloat16)
    run_and_check(s, gate=gate)


@pytest.mark.parametrize("qlens", [
    [700], [300, 1, 0, 170], [200, 1, 1, 3, 0, 171],            # items of a sequence: many
    [1] * 33, [20] * 33,                                        # more sequences than a warp
    [1] * 1100, [1] * 1050 + [200], [33] + [1] * 1050,          # than the plan keeps
])
def test_plans(qlens):
    g = torch.Generator().manual_seed(len(qlens))
    lens = [n + int(torch.randint(0, 40, (1,), generator=g)) if n else 0 for n in qlens]
    run_and_check(make(73, lens, qlens, 1, 64, 8, 16))


@pytest.mark.parametrize("H,KV,D,qlens", [(128, 1, 64, [1, 2, 5]), (128, 1, 256, [1, 3]), (127, 1, 128, [1, 4])])
def test_as_many_heads_per_key_as_allowed(H, KV, D, qlens):
    run_and_check(make(74, [200 + 31 * n for n in qlens], qlens, KV, D, H, 64))


@pytest.mark.parametrize("H,KV,D", [(8, 1, 64), (10, 2, 40), (8, 1, 128), (8, 1, 136)])
@pytest.mark.parametrize("opts", [{}, dict(window=50, softcap=8.0)])
def test_rows_between_the_kernels(H, KV, D, opts):
    """17 to 32 rows of a key/value head, and the first count beyond."""
    run_and_check(make(79, [500, 3, 33, 2100], [4, 3, 0, 4], KV, D, H, 16), **opts)
    run_and_check(make(80, [500, 5, 2100], [5, 5, 1], KV, D, H, 16, prefix=40), **opts)


@pytest.mark.parametrize("qlens,bound", [([1, 1, 1], 2), ([1, 2, 1], 4), ([1, 2, 3], 700), ([30, 2], 5000)])
def test_bounds_above_the_lengths(qlens, bound):
    lens = [400 + 97 * i for i in range(len(qlens))]
    run_and_check(make(75, lens, qlens, 2, 128, 8, 16), single=False, max_q=bound)


def test_two_calls_at_once_and_a_workspace_used_again():
    """Calls on two streams with a workspace each, in turns of different shapes."""
    import nvfp4

    sets = [make(76, [3000, 17], [1, 1], 2, 128, 8, 16), make(77, [900, 500], [300, 260], 2, 128, 8, 64),
            make(78, [700] * 6, [1] * 6, 2, 128, 8, 16, prefix=900)]
    cfg = nvfp4.AttentionConfig(8, 2, 128, causal=True)
    batches = [batch_of(s) for s in sets]
    queries = [s["q"].cuda() for s in sets]
    alone = [nvfp4.paged_attention(q, s["cache"], b, cfg) for s, b, q in zip(sets, batches, queries)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    sizes = [nvfp4.attention_workspace(cfg, b).numel() for b in batches]
    spaces = [torch.full((max(sizes),), 0xff, dtype=torch.uint8, device="cuda") for _ in streams]
    torch.cuda.synchronize()
    got = []
    for turn in range(6):
        for i, (st, ws) in enumerate(zip(streams, spaces)):
            with torch.cuda.stream(st):
                k = (turn + i) % 3
                got.append((k, nvfp4.paged_attention(queries[k], sets[k]["cache"], batches[k], cfg, workspace=ws)))
    torch.cuda.synchronize()
    for k, o in got:
        assert torch.equal(o, alone[k])


@pytest.mark.parametrize("qlens", [[1, 1, 1], [2, 1, 40]])
def test_offsets_beyond_32_bits(qlens):
    """The last pages of a cache of 2.3 G elements, rows 2^30 elements apart in
    q: the results of a small cache and packed rows, bit for bit."""
    import nvfp4

    H, KV, D, page, far = 8, 4, 128, 64, 70000
    T, lens = sum(qlens), [n + 130 for n in qlens]
    g = torch.Generator().manual_seed(81)
    rows = lambda heads: torch.randn(T, heads, D, generator=g).to(torch.bfloat16).cuda()
    q, k, v = rows(H), rows(KV), rows(KV)
    small = [torch.randn(12, page, KV, D, generator=g).to(torch.bfloat16).cuda() for _ in range(2)]
    big = [torch.empty(far, page, KV, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for s, b in zip(small, big):
        b[-12:] = s
    table = torch.randperm(12, generator=g)[:9].reshape(3, 3).to(torch.int32).cuda()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    starts = i32([0, qlens[0], qlens[0] + qlens[1], T])
    apart = torch.empty(min(T, 3) * 2 ** 30, dtype=torch.bfloat16, device="cuda")
    q_far = apart.as_strided((T, H, D), (2 ** 30 if T <= 3 else 2 ** 26, D, 1))
    q_far.copy_(q)
    cfg = nvfp4.AttentionConfig(H, KV, D, causal=True)
    got = []
    for cache, pages, queries in ((small, table, q), (big, table + (far - 12), q_far)):
        cache = nvfp4.PagedKVCache(*cache)
        batch = nvfp4.AttentionBatch(i32(lens), pages, q_start=starts, num_tokens=T, max_q_len=max(qlens))
        turned = nvfp4.kv_append(queries, k, v, cache, batch, q_out=queries)
        got.append((turned.clone(), nvfp4.paged_attention(turned, cache, batch, cfg)))
    torch.cuda.synchronize()
    for s, b in zip(small, big):
        assert torch.equal(s, b[-12:])
    assert torch.equal(*(x[0] for x in got)) and torch.equal(*(x[1] for x in got))


@pytest.mark.parametrize("D", [8, 24, 72, 120, 200, 248])
@pytest.mark.parametrize("qlens", [[1, 1, 1], [1, 70, 6]])
def test_head_sizes_that_fill_no_tile(D, qlens):
    for prefix in (0, 33):
        s = make(82, [n + 150 for n in qlens], qlens, 2, D, 6, 16, prefix=prefix)
        gate = torch.randn(s["T"], s["H"], D, generator=s["g"]).to(torch.bfloat16)
        run_and_check(s, gate=gate, window=100)
        run_and_check(s, causal=False)


def test_overlapping_token_ranges_beyond_the_bounds():
    """Every other sequence claims all tokens: more work than the counts allow
    for.  Nothing is followed out of range, and the next call is right."""
    import nvfp4
    from nvfp4 import _lib

    B, T, H, KV, D = 2300, 16384, 32, 4, 64
    k, v = (torch.zeros(8, 64, KV, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table = torch.zeros(1, dtype=torch.int32, device="cuda").expand(B, 940).contiguous()
    starts = torch.tensor([0, T] * (B // 2) + [0], dtype=torch.int32, device="cuda")
    batch = nvfp4.AttentionBatch(torch.full((B,), 60000, dtype=torch.int32, device="cuda"), table, q_start=starts,
                                 num_tokens=T, max_q_len=16)
    q = torch.zeros(T, H, D, dtype=torch.bfloat16, device="cuda")
    nvfp4.paged_attention(q, nvfp4.PagedKVCache(k, v), batch, nvfp4.AttentionConfig(H, KV, D, causal=False))
    torch.cuda.synchronize()
    assert _lib.load().nvfp4_device_status() == 0
    run_and_check(make(83, [300, 20], [1, 20], 2, 64, 8, 16))
