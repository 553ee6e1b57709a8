"""The attention side of a decoder layer on a paged cache, and the layer's decode step around the sparse MoE block.

The reference leaves attention, norms and the cache to its models' torch code (``modeling_mixtral.py``); here
they run beside the compact3 projections (``qlinear.Compact3Linear``) and the block (``moe.TrisSparseMoeBlock``):

* ``rotary_tables``      cosines and sines of the positions;
* ``PagedKVCache``       the pool of pages of one layer, fp16, bf16 or e4m3 with a scale per token and kv head, and, where
                         it is asked for, the sums of the attention weights and the eviction by them;
* ``TrisPagedAttention`` projections, rotation and append, attention, output projection;
* ``TrisDecoderLayer``   norm, attention, norm with the residual's addition, MoE block.

Block tables and lengths are the caller's (one pair serves all layers); every step takes them from device tensors, so
a captured decode step is replayed with other lengths and tables.  Rotary positions are the tokens' places in the cache,
or the caller's: on several axes for images, and for every token after an eviction, which leaves a sequence shorter than
its positions.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from . import ext
from .qlinear import run_compact3_qkv_block_gr_forward


def rotary_tables(rotary_dim: int, positions: int, theta: float = 10000.0, device="cuda"):
    """(cos, sin) fp32 [positions, rotary_dim / 2] of position * theta^(-2 i / rotary_dim).  The angles are taken in 64
    bits: in 32, those of far positions are off by more than a table entry's rounding."""
    if rotary_dim < 16 or rotary_dim % 16:
        raise ValueError("rotary_dim must be a positive multiple of 16")
    freq = float(theta) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * freq[None]
    return angle.cos().to(torch.float32), angle.sin().to(torch.float32)


class PagedKVCache:
    """One layer's pool of pages: k and v [pages, kv_heads, page_size, head_dim] of dtype (float16, bfloat16, or
    float8_e4m3fn with k_scale and v_scale fp32 [pages, kv_heads, page_size]).  A 16-bit cache takes activations of
    its own type: under ``TrisPagedAttention``, whose projections are fp16, a cache is float16 or float8_e4m3fn.
    Which pages a sequence has is the block table's matter; a page's contents count only below the lengths given with
    it.  weight_sum: None, or after ``track_weights`` fp32 [batch, kv_heads, positions], the attention weights that each
    place has had, row b for the block table's row b; a caller that gives row b to a new sequence sets it to zero, and one
    that moves a sequence to another row moves its sums too."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype: torch.dtype = torch.float16,
                 device="cuda"):
        if head_dim not in ext.PAGED_HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {ext.PAGED_HEAD_DIMS}")
        if dtype not in (torch.float16, torch.bfloat16, torch.float8_e4m3fn):
            raise ValueError("a cache is float16, bfloat16 or float8_e4m3fn")
        shape = (pages, kv_heads, page_size, head_dim)
        self.k, self.v = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
        self.k_scale = self.v_scale = self.weight_sum = None
        if dtype == torch.float8_e4m3fn:
            self.k_scale, self.v_scale = (torch.empty(shape[:3], dtype=torch.float32, device=device) for _ in range(2))

    def track_weights(self, batch: int, positions: int) -> None:
        """From now on ``attend`` sums the attention weights of block tables of up to `batch` rows and `positions`
        positions (max_pages * page_size), from zero."""
        self.weight_sum = torch.zeros((batch, self.k.size(1), positions), dtype=torch.float32, device=self.k.device)

    def _sums(self, block_table):
        """The sums of a block table's rows: of fewer than `batch`, the first ones'."""
        if self.weight_sum is None or not isinstance(block_table, torch.Tensor) or block_table.ndim != 2:
            return self.weight_sum
        rows = block_table.size(0)
        return self.weight_sum if rows >= self.weight_sum.size(0) else self.weight_sum[:rows]

    def append(self, q, k, v, cos, sin, block_table, seq_lens, query_start=None, positions=None, sections=None,
               interleaved=False):
        """ext.rotary_append_paged on this pool: the rotated queries."""
        return ext.rotary_append_paged(q, k, v, cos, sin, self.k, self.v, block_table, seq_lens, query_start,
                                       k_scale=self.k_scale, v_scale=self.v_scale, positions=positions,
                                       sections=sections, interleaved=interleaved)

    def attend(self, q, block_table, seq_lens, scale=None, window=0):
        """ext.paged_attention_decode on this pool."""
        return ext.paged_attention_decode(q, self.k, self.v, block_table, seq_lens, scale, window,
                                          k_scale=self.k_scale, v_scale=self.v_scale,
                                          weight_sum=self._sums(block_table))

    def evict(self, block_table, seq_lens, budget, limit=None, sink=0, recent=0):
        """ext.paged_cache_evict on this pool: (new lengths, kept positions).  With one pair of tables for all layers,
        every layer evicts by the old lengths; then seq_lens takes the new ones, which are the same for each."""
        if self.weight_sum is None:
            raise RuntimeError("evict: the cache has no sums of attention weights (track_weights)")
        return ext.paged_cache_evict(self.k, self.v, block_table, seq_lens, self._sums(block_table), budget, limit, sink,
                                     recent, k_scale=self.k_scale, v_scale=self.v_scale)


class TrisPagedAttention(nn.Module):
    """Attention over compact3 projections and a paged cache.  q_proj, k_proj, v_proj and o_proj: Compact3Linear (fp16
    inputs and outputs).  q_norm, k_norm: norm weights of [head_dim] (each head) or of the whole projection
    ([heads * head_dim]), or None.  cos, sin: rotary_tables.  window: positions that a token attends to (0: all).
    sections, interleaved: the pairs of each rotary axis, for steps that give positions of several
    (ext.rotary_append_paged)."""

    def __init__(self, q_proj, k_proj, v_proj, o_proj, num_heads: int, num_kv_heads: int, head_dim: int,
                 cos: torch.Tensor, sin: torch.Tensor, q_norm: torch.Tensor | None = None,
                 k_norm: torch.Tensor | None = None, norm_eps: float = 1e-6, window: int = 0,
                 scale: float | None = None, sections: tuple | None = None, interleaved: bool = False):
        super().__init__()
        if num_heads % num_kv_heads:
            raise ValueError("num_heads must be a multiple of num_kv_heads")
        for name, proj, width in (("q_proj", q_proj, num_heads * head_dim), ("k_proj", k_proj, num_kv_heads * head_dim),
                                  ("v_proj", v_proj, num_kv_heads * head_dim)):
            if proj.outfeatures != width:
                raise ValueError(f"{name} must have {width} outputs")
        if sections is not None and sum(sections) != cos.size(1):
            raise ValueError("sections must add up to the columns of cos")
        if o_proj.infeatures != num_heads * head_dim:
            raise ValueError(f"o_proj must have {num_heads * head_dim} inputs")
        self.q_proj, self.k_proj, self.v_proj, self.o_proj = q_proj, k_proj, v_proj, o_proj
        self.num_heads, self.num_kv_heads, self.head_dim = num_heads, num_kv_heads, head_dim
        self.norm_eps, self.window, self.scale = norm_eps, window, scale
        self.sections, self.interleaved = None if sections is None else tuple(sections), interleaved
        for name, t in (("cos", cos), ("sin", sin), ("q_norm", q_norm), ("k_norm", k_norm)):
            self.register_buffer(name, t, persistent=False)

    def _normed(self, x, weight):
        """x [tokens, heads, head_dim] under a norm of each head or of the whole row."""
        if weight is None:
            return x
        rows = x if weight.numel() == self.head_dim else x.view(x.size(0), x.size(1) * x.size(2))
        return ext.rms_norm(rows, weight, self.norm_eps).view(x.shape)

    @torch.no_grad()
    def append(self, x16: torch.Tensor, cache: PagedKVCache, block_table: torch.Tensor, seq_lens: torch.Tensor,
               query_start: torch.Tensor | None = None, positions: torch.Tensor | None = None) -> torch.Tensor:
        """Projects new tokens x16 [tokens, hidden] (a decode step's, or prompts' with query_start), appends their keys
        and values and returns the rotated queries [tokens, num_heads, head_dim].  positions int32 [axes, tokens] (or
        [tokens], the same on every axis): rotary positions other than the tokens' places."""
        fused = run_compact3_qkv_block_gr_forward(self.q_proj, self.k_proj, self.v_proj, x16)
        q, k, v = fused if fused is not None else (self.q_proj(x16), self.k_proj(x16), self.v_proj(x16))
        q, k, v = (t.view(t.size(0), t.size(1) // self.head_dim, self.head_dim) for t in (q, k, v))
        q, k = self._normed(q, self.q_norm), self._normed(k, self.k_norm)
        if positions is None:
            return cache.append(q, k, v, self.cos, self.sin, block_table, seq_lens, query_start)
        several = positions.ndim == 2 and positions.size(0) > 1
        return cache.append(q, k, v, self.cos, self.sin, block_table, seq_lens, query_start, positions,
                            self.sections if several else None, self.interleaved and several)

    @torch.no_grad()
    def decode(self, x16: torch.Tensor, cache: PagedKVCache, block_table: torch.Tensor, seq_lens: torch.Tensor,
               positions: torch.Tensor | None = None) -> torch.Tensor:
        """One new token a sequence, x16 fp16 [batch, hidden] (seq_lens counts it; positions as append takes them): the
        layer's attention, fp16 [batch, hidden]."""
        q = self.append(x16, cache, block_table, seq_lens, positions=positions)
        y = cache.attend(q, block_table, seq_lens, self.scale, self.window)
        return self.o_proj(y.view(y.size(0), self.num_heads * self.head_dim))


class TrisDecoderLayer(nn.Module):
    """A decoder layer's decode step: attention and MoE block, each behind a norm that adds what came before it to the
    residual stream (modeling_mixtral.py's decoder layer, its two additions moved into the norms that follow them)."""

    def __init__(self, attention: TrisPagedAttention, block, input_norm: torch.Tensor, post_norm: torch.Tensor,
                 norm_eps: float = 1e-5):
        super().__init__()
        self.attention, self.block, self.norm_eps = attention, block, norm_eps
        self.register_buffer("input_norm", input_norm, persistent=False)
        self.register_buffer("post_norm", post_norm, persistent=False)

    @torch.no_grad()
    def decode(self, x: torch.Tensor, residual: torch.Tensor | None, cache: PagedKVCache, block_table: torch.Tensor,
               seq_lens: torch.Tensor, positions: torch.Tensor | None = None):
        """x [batch, hidden]: the layer below's output (the embedding in the first layer, with residual None), residual
        the stream without it, both in the model dtype; positions as TrisPagedAttention.append takes them.  Returns the
        same pair for the layer above; after the last layer the stream is x + residual, which the final
        rms_norm(x, weight, eps, residual=residual) adds."""
        if residual is None:
            residual = x
            h = ext.rms_norm(x, self.input_norm, self.norm_eps, out_dtype=torch.float16)
        else:
            h, residual = ext.rms_norm(x, self.input_norm, self.norm_eps, residual=residual, out_dtype=torch.float16)
        y = self.attention.decode(h, cache, block_table, seq_lens, positions)
        h, residual = ext.rms_norm(y, self.post_norm, self.norm_eps, residual=residual, out_dtype=residual.dtype)
        out, _ = self.block(h.unsqueeze(0))
        return out.squeeze(0), residual
