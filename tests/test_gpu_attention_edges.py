"""What paged_attention, kv_append, norm_residual and AttentionLayer must also
get right: large caps, distances beyond 2^24, values that are not finite, rows
in no sequence, loops beyond their first turn."""
import math

import pytest
import torch

import attention_ref as ref
from test_gpu_attention import append_case, batch_of, make, run_and_check, test_norm_residual as norm_case

pytestmark = pytest.mark.gpu


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
