"""AttentionLayer: rows in no sequence, the heads' norms of a loaded layer, and
weights that are stacked on another stream."""
import math
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import st_fixtures as F
from test_gpu_attention_layer import build, close, loaded, reference
from test_gpu_loader import moe_checkpoint
from nvfp4.weight_loader import SafetensorsModel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,gated,res", [(128, False, torch.bfloat16), (256, True, torch.float32)])
def test_rows_in_no_sequence_get_no_attention(O, D, gated, res):
    """A batch padded behind its last sequence: its rows' residual is what it
    would be without the layer, whatever the memory held before."""
    import nvfp4

    H, KV, d_model, lens, pad = 4, 1, 512, [20, 33], 11
    att, m = build(O, 17, H, KV, D, d_model, gated, 64)
    g = torch.Generator().manual_seed(5)
    T = sum(lens)
    cache = nvfp4.PagedKVCache.empty(8, 16, KV, D)
    cache.k.fill_(math.nan)
    cache.v.fill_(math.nan)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    batch = nvfp4.AttentionBatch(i32(lens), i32([[5, 2, 0], [1, 7, 3]]), q_start=i32([0, lens[0], T]),
                                 num_tokens=T + pad, max_q_len=max(lens))
    x = torch.randn(T + pad, d_model, generator=g).to(res)
    ws = nvfp4.attention_workspace(att.config, batch)
    for _ in range(2):
        spoilt = torch.full((T + pad, H, D), math.nan, dtype=torch.bfloat16, device="cuda")
        del spoilt  # its memory is the next of that size
        r, y = att.step(None, x.cuda(), cache, batch, workspace=ws)
        assert torch.equal(r[T:].cpu(), x[T:]) and torch.isfinite(y[T:]).all()
        past = [[torch.zeros(0, KV, D, dtype=torch.float64) for _ in range(2)] for _ in lens]
        want = [reference(m, z, p) for z, p in zip(x[:T].double().split(lens), past)]
        close(r[:T], torch.cat([w[0] for w in want]))
        close(y[:T], torch.cat([w[1] for w in want]))


@pytest.mark.parametrize("normed", [True, False])
def test_the_heads_norms_of_a_loaded_layer_are_used(tmp_path, normed):
    """self_attn.q_norm and k_norm of a checkpoint that has them reach the
    layer; a checkpoint without them loads as before."""
    import nvfp4

    E, d_model, H, KV, D = 4, 256, 4, 1, 128
    moe_checkpoint(tmp_path / "experts.safetensors", E, d_model, 128, 256, seed=31)
    rng = np.random.default_rng(32)
    g = torch.Generator().manual_seed(33)
    lp, t = "model.layers.0", {}
    for p, (n, k) in {"q_proj": (H * D, d_model), "k_proj": (KV * D, d_model), "v_proj": (KV * D, d_model),
                      "o_proj": (d_model, H * D)}.items():
        w, sf = F.rand_linear(rng, n, k)
        F.nvfp4_linear(t, f"{lp}.self_attn.{p}", w, sf, ws2=np.float32(1e-3))
    vec = lambda n: (1 + 0.3 * torch.randn(n, generator=g)).to(torch.bfloat16)
    t[f"{lp}.input_layernorm.weight"], t[f"{lp}.post_attention_layernorm.weight"] = vec(d_model), vec(d_model)
    qn, kn = vec(D), vec(D).float()
    if normed:
        t[f"{lp}.self_attn.q_norm.weight"], t[f"{lp}.self_attn.k_norm.weight"] = qn, kn
    F.save(tmp_path / "attn.safetensors", t)
    model = SafetensorsModel.from_files([str(tmp_path / "attn.safetensors"), str(tmp_path / "experts.safetensors")])
    layer = nvfp4.load_qwen35_layer(model, 0, E)
    model.close()
    weights = nvfp4.AttentionWeights.from_layer(layer)
    if not normed:
        assert weights.q_norm is None and weights.k_norm is None
        return
    assert torch.equal(weights.q_norm.cpu(), qn) and torch.equal(weights.k_norm.cpu(), kn.to(torch.bfloat16))
    other = nvfp4.AttentionWeights.from_layer(layer, k_norm=qn)  # the caller's come first
    assert torch.equal(other.q_norm.cpu(), qn) and torch.equal(other.k_norm.cpu(), qn)


def test_weights_stacked_on_another_stream_are_ready(O):
    """from_layer on a stream that is busy: what the caller's stream reads next
    is the stacked weights, and nothing that it still uses is overwritten."""
    import nvfp4

    H, KV, D, d_model = 8, 2, 128, 512
    layer, m = {}, {}
    rng = np.random.default_rng(41)
    for p, (n, k) in {"q_proj": (H * D, d_model), "k_proj": (KV * D, d_model), "v_proj": (KV * D, d_model),
                      "o_proj": (d_model, H * D)}.items():
        layer[p], m[p] = loaded(O, rng, n, k, p != "k_proj")
    one = torch.ones(d_model, dtype=torch.bfloat16).view(torch.uint8).numpy()
    layer = SimpleNamespace(**layer, input_layernorm=one, post_attn_layernorm=one, q_norm=torch.full((D,), 2.0),
                            k_norm=None)
    parts = lambda w: (*w.in_proj[1:], w.in_proj[0].weight_scale_2_rows, w.q_norm, w.input_norm)
    want = [t.cpu() for t in parts(nvfp4.AttentionWeights.from_layer(layer))]
    assert torch.equal(want[0], torch.cat([p.packed_weights.cpu() for p in (layer.q_proj, layer.k_proj, layer.v_proj)]))
    for side in (torch.cuda.Stream(), torch.cuda.Stream()):
        for stream in (side, side.cuda_stream):
            source = torch.arange(want[0].numel(), device="cuda") % 251
            torch.cuda.synchronize()
            spare = torch.empty_like(source, dtype=torch.uint8)
            torch.cuda._sleep(20_000_000)  # the caller's stream is busy,
            spare.copy_(source)
            kept = spare.clone()           # with memory of the weights' size
            del spare
            with torch.cuda.stream(side):
                torch.cuda._sleep(20_000_000)  # and so is the other one
            weights = nvfp4.AttentionWeights.from_layer(layer, stream=stream)
            got = [t.clone() for t in parts(weights)]
            torch.cuda.synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a.cpu(), b)
            assert torch.equal(kept.cpu(), source.cpu().to(torch.uint8))
