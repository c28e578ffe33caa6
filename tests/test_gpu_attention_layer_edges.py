"""AttentionLayer: rows in no sequence, the heads' norms of a loaded layer, and
weights that are stacked on another stream."""
import math
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import st_fixtures as F
from test_gpu_attention_layer import build, close, reference
from test_gpu_loader import moe_checkpoint
from nvfp4.weight_loader import SafetensorsModel

pytestmark = pytest.mark.gpu


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
