"""A softmax-attention layer with NVFP4 projections, for prompts and single
tokens: norm and residual, one input projection, the cache append with norm
and rotation, attention over the paged cache, output projection.

The projections are the reference's q/k/v/o_proj (nvfp4/weight_loader.mojo:
776-893), which it loads and does not multiply."""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from .attention import AttentionBatch, AttentionConfig, PagedKVCache, Rotary, kv_append, paged_attention
from .config import NvFp4Linear
from .moe import _row_scales, stack_rows
from .nvfp4_gemm_gpu import _u8, nvfp4_linear
from .norm import norm_residual


def _bf16_vector(raw, device) -> torch.Tensor:
    """A norm's weight: a tensor, or the raw bytes of a bf16 one."""
    if not torch.is_tensor(raw):
        raw = torch.from_numpy(raw.copy()).view(torch.bfloat16).reshape(-1)
    return raw.to(device, torch.bfloat16).contiguous()


@dataclass
class AttentionWeights:
    """in_proj: (NvFp4Linear, packed weights, blockscales) of the rows [q; k;
    v], q's head by head; with an output gate each head's rows are [query;
    gate].  out: the same of the output projection.  Norm weights bf16;
    q_norm and k_norm [head_dim] or None."""

    in_proj: tuple
    out: tuple
    input_norm: torch.Tensor
    post_norm: torch.Tensor
    q_norm: Optional[torch.Tensor] = None
    k_norm: Optional[torch.Tensor] = None

    @classmethod
    def from_layer(cls, layer, q_norm=None, k_norm=None, stream=None) -> "AttentionWeights":
        """From a layer of `load_qwen35_layer`: q, k and v stacked into one
        matrix (one launch instead of three), each one's input_scale folded
        into its rows' weight_scale_2 (the product is the same).  q_norm and
        k_norm None: the layer's own, where it has them."""
        device = layer.q_proj.packed_weights.device
        with torch.cuda.device(device):
            here = torch.cuda.current_stream()
            if stream is None:
                stream = here
            elif not isinstance(stream, torch.cuda.Stream):
                stream = torch.cuda.ExternalStream(int(stream), device=device)
            # Everything is made on `stream`, after what the caller has under way,
            # and before what comes on the caller's own stream, where the layer runs.
            stream.wait_stream(here)
            with torch.cuda.stream(stream):
                w = cls._stack(layer, device, q_norm, k_norm)
            here.wait_stream(stream)
            for t in (w.in_proj[0].weight_scale_2_rows, *w.in_proj[1:], w.input_norm, w.post_norm, w.q_norm, w.k_norm):
                if t is not None:
                    t.record_stream(here)
        return w

    @classmethod
    def _stack(cls, layer, device, q_norm, k_norm) -> "AttentionWeights":
        parts = (layer.q_proj, layer.k_proj, layer.v_proj)
        w = stack_rows([p.packed_weights for p in parts])
        sf = stack_rows([_u8(p.blockscales) for p in parts])
        rows = [_row_scales(p.weight_scale_2 if p.weight_scale_2_rows is None else p.weight_scale_2_rows,
                            p.out_features, p.input_scale).to(device) for p in parts]
        lin = NvFp4Linear(parts[0].in_features, w.shape[0], weight_scale_2_rows=torch.cat(rows))
        q_norm, k_norm = (getattr(layer, n, None) if w is None else w
                          for n, w in (("q_norm", q_norm), ("k_norm", k_norm)))
        o = layer.o_proj
        vec = lambda x: None if x is None else _bf16_vector(x, device)
        return cls((lin, w, sf), (o.to_linear(), o.packed_weights, o.blockscales),
                   vec(layer.input_layernorm), vec(layer.post_attn_layernorm), vec(q_norm), vec(k_norm))


class AttentionLayer:
    """One layer.  `step` takes the block output before it and the residual
    stream and returns the residual and the input of the block after it:

        r, h = norm(x + residual);  r, y = norm(r + o_proj(attention(h)))
    """

    def __init__(self, weights: AttentionWeights, config: AttentionConfig, rotary: Optional[Rotary] = None,
                 gated: bool = False, norm_eps: float = 1e-6, norm_offset: float = 0.0):
        self.w, self.config, self.rotary, self.gated = weights, config, rotary, gated
        self.eps, self.offset = norm_eps, norm_offset
        H, KV, D = config.num_heads, config.num_kv_heads, config.head_dim
        if weights.in_proj[0].out_features != (H * (2 if gated else 1) + 2 * KV) * D:
            raise ValueError("the input projection's rows do not match the heads")
        if weights.out[0].in_features != H * D:
            raise ValueError("the output projection's columns do not match the heads")

    def attention(self, h: torch.Tensor, cache: PagedKVCache, batch: AttentionBatch,
                  positions: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
        """h bf16 [T, d_model], normed -> o_proj(attention) bf16 [T, d_model];
        this step's keys and values go into the cache.  Rows in no sequence
        (a padded batch) have an attention of 0."""
        c = self.config
        H, KV, D, T = c.num_heads, c.num_kv_heads, c.head_dim, h.shape[0]
        x = nvfp4_linear(*self.w.in_proj, h)
        nq = H * (2 if self.gated else 1)
        q, k, v = x.view(T, nq + 2 * KV, D).split([nq, KV, KV], dim=1)
        gate = None
        if self.gated:
            heads = x[:, :nq * D].view(T, H, 2, D)
            q, gate = heads[:, :, 0], heads[:, :, 1]
        # (Append and attention leave rows in no sequence as they are.)
        q_out = None if batch.tensors[2] is None else torch.zeros(T, H, D, dtype=torch.bfloat16, device=x.device)
        q = kv_append(q, k, v, cache, batch, rotary=self.rotary, positions=positions, q_norm=self.w.q_norm,
                      k_norm=self.w.k_norm, norm_eps=self.eps, norm_offset=self.offset, q_out=q_out)
        a = paged_attention(q, cache, batch, c, gate=gate, out=q, workspace=workspace)
        return nvfp4_linear(*self.w.out, a.view(T, H * D))

    def step(self, x: Optional[torch.Tensor], residual: torch.Tensor, cache: PagedKVCache, batch: AttentionBatch,
             positions: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None
             ) -> Tuple[torch.Tensor, torch.Tensor]:
        """x bf16 [T, d_model]: the output of the block before (None: the
        first block; residual is its input), residual bf16 or fp32, updated in
        place.  Returns (residual, y), y bf16 the normed input of the block
        that follows (an MoE layer's)."""
        if x is None:
            _, h = norm_residual(residual, pre_weight=self.w.input_norm, eps=self.eps, weight_offset=self.offset,
                                 residual_out=residual)
        else:
            _, h = norm_residual(x, residual, pre_weight=self.w.input_norm, eps=self.eps,
                                 weight_offset=self.offset, residual_out=residual)
        a = self.attention(h, cache, batch, positions, workspace)
        return norm_residual(a, residual, pre_weight=self.w.post_norm, eps=self.eps, weight_offset=self.offset,
                             residual_out=residual)


__all__ = ["AttentionWeights", "AttentionLayer"]
