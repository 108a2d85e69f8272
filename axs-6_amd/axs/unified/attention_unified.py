"""Attention without the score matrix, and a decoder's self-attention on it.

``axs_attention_unified`` computes softmax(scale q k^T + mask) v and its
gradients on the matrix cores, a tile of scores at a time; the backward makes
the probabilities again from one number a row.  Unlike
``AXSMultiheadAttentionUnified`` (the reference's module,
``axs/unified/modules_unified.py:192-264``) it does not fake-quantize the
probabilities.  ``AXSCausalSelfAttentionUnified`` joins it with the quantized
projections, rotary positions and the 8-bit cache.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from axs import _lib
from axs.core import DEFAULT_BLOCK_SIZE
from axs.unified.functional_unified import axs_linear_group_unified
from axs.unified.kv_cache_unified import (
    AXSKVCacheUnified,
    axs_cache_append_unified,
    axs_cache_attention_unified,
    axs_cache_shared_attention_unified,
)
from axs.unified.modules_unified import AXSLinearUnified
from axs.unified.rotary_unified import axs_rotary_unified


def axs_attention_unified(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    mask: torch.Tensor | None = None,
    causal: bool = False,
    scale: float | None = None,
) -> torch.Tensor:
    """softmax(scale q k^T + mask) v -> (B, Tq, Hq, D).

    ``q`` (B, Tq, Hq, D), ``k`` and ``v`` (B, Tk, Hkv, D), Hq a multiple of Hkv
    (query head h reads key head h // (Hq / Hkv)), D up to 128, float32, bfloat16 or
    float16 in any layout whose heads' values are adjacent ((B, H, T, D) tensors:
    pass ``x.transpose(1, 2)``).  ``causal``: query i sees keys j <= i + Tk - Tq.
    ``mask`` broadcasts to (B, Hq, Tq, Tk): bool, True where a query sees a key, or
    values added to the scores, -inf where it does not; no gradient.  A query that
    sees no key gives 0.  ``scale`` is 1 / sqrt(D) if None, else positive.

    A result that is not finite is made again pair by pair (places that a query does not
    see have no part in it), which takes much longer.

    Scores, softmax and sums are float32; for 16-bit operands the probabilities
    (and, in the backward, their gradients) are rounded to the operands' type for
    the second product.  Gradients for q, k and v, summed in a fixed order.
    """
    return _lib.ext().attention(q, k, v, mask, causal, scale)


class AXSCausalSelfAttentionUnified(nn.Module):
    """A decoder's self-attention: NF5-quantized projections, rotary positions,
    causal attention of grouped heads; :meth:`decode` answers from the 8-bit cache.

    ``num_kv_heads`` key heads are shared by groups of the ``num_heads`` query heads
    (None: each has its own)."""

    def __init__(
        self,
        embed_dim: int,
        num_heads: int,
        num_kv_heads: int | None = None,
        bias: bool = True,
        block_size: int = DEFAULT_BLOCK_SIZE,
    ) -> None:
        super().__init__()
        num_kv_heads = num_heads if num_kv_heads is None else num_kv_heads
        if embed_dim % num_heads or num_heads % num_kv_heads:
            raise ValueError(f"{num_heads} heads do not divide {embed_dim} values, or {num_kv_heads} key heads them")
        self.embed_dim, self.num_heads, self.num_kv_heads = embed_dim, num_heads, num_kv_heads
        self.head_dim = embed_dim // num_heads
        self.block_size = block_size
        kv = num_kv_heads * self.head_dim
        self.q_proj = AXSLinearUnified(embed_dim, embed_dim, bias=bias, block_size=block_size)
        self.k_proj = AXSLinearUnified(embed_dim, kv, bias=bias, block_size=block_size)
        self.v_proj = AXSLinearUnified(embed_dim, kv, bias=bias, block_size=block_size)
        self.out_proj = AXSLinearUnified(embed_dim, embed_dim, bias=bias, block_size=block_size)

    def _heads(self, x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """Queries, keys and values: one grouped linear where the three projections are
        quantized ones of the same settings, else one by one -- also when a projection
        has hooks, which see only calls of the module itself."""
        p = (self.q_proj, self.k_proj, self.v_proj)
        grouped = (all(type(m) is AXSLinearUnified for m in p)
                   and not any(m._warmup_active or m._forward_hooks or m._forward_pre_hooks for m in p)
                   and len({(m.block_size, m.quantize_input, m.quantize_grad) for m in p}) == 1)
        if grouped:
            m = p[0]
            y = axs_linear_group_unified(x, [l.weight for l in p], [l.bias for l in p], m.block_size,
                                         m.quantize_input, m.quantize_grad)
        else:
            y = tuple(m(x) for m in p)
        B, T = x.shape[:2]
        return tuple(t.reshape(B, T, -1, self.head_dim) for t in y)

    def forward(self, x: torch.Tensor, table: torch.Tensor, positions: torch.Tensor | None = None) -> torch.Tensor:
        """``x`` (B, T, embed_dim), whole sequences; ``table`` and ``positions`` as in
        :func:`axs_rotary_unified`."""
        q, k, v = self._heads(x)
        q, k = axs_rotary_unified(q, k, table, positions)
        return self.out_proj(axs_attention_unified(q, k, v, causal=True).flatten(2))

    def new_cache(self, batch: int, max_tokens: int, dtype: torch.dtype = torch.float32,
                  device: torch.device | str = "cuda") -> AXSKVCacheUnified:
        """An empty cache of this layer's heads."""
        return AXSKVCacheUnified.empty(batch, self.num_kv_heads, self.head_dim, max_tokens, dtype, device)

    def decode(self, x: torch.Tensor, table: torch.Tensor, cache: AXSKVCacheUnified, starts: torch.Tensor,
               prefix: AXSKVCacheUnified | None = None, prefix_lengths: torch.Tensor | None = None) -> torch.Tensor:
        """``x`` (B, T, embed_dim): tokens ``starts[b]``.. of each sequence, a prompt's
        or the next one.  They join the cache and attend over it; no gradient.

        ``prefix``, a cache of P sequences of ``prefix_lengths`` (P) tokens: sequence b goes on from
        prefix b // (B / P), its tokens' places counted from the prefix's end, and attends over
        both (:func:`axs_cache_shared_attention_unified`)."""
        if (prefix is None) != (prefix_lengths is None):
            raise ValueError("a prefix and its lengths come together")
        with torch.no_grad():
            q, k, v = self._heads(x)
            places = starts
            if prefix is not None:
                P = prefix_lengths.numel()
                if P == 0 or x.shape[0] % P or prefix.k_codes.shape[0] != P:
                    raise ValueError(f"{x.shape[0]} sequences do not divide among {P} prefixes, or a cache of "
                                     f"{prefix.k_codes.shape[0]} does not hold them")
                places = starts + prefix_lengths.repeat_interleave(x.shape[0] // P, output_size=x.shape[0])
            positions = places[:, None] + torch.arange(x.shape[1], device=x.device)
            q, k = axs_rotary_unified(q, k, table, positions)
            axs_cache_append_unified(cache, k, v, starts)
            if prefix is None:
                out = axs_cache_attention_unified(q, cache, starts + x.shape[1])
            else:
                out = axs_cache_shared_attention_unified(q, prefix, prefix_lengths, cache, starts + x.shape[1])
            return self.out_proj(out.flatten(2))
