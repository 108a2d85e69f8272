"""Keys and values in 8 bits, with a scale for each block of 32 tokens and head.

A block of one head holds code * scale, scale = max |x| / 127 over the block's
tokens (float32) and code = round(x / scale).  The block that is not full yet
is held raw beside its codes and quantized anew when a token joins it, so the
cache depends on the tokens alone and not on the calls that brought them.
The reference has no cache.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from axs import _lib

CACHE_BLOCK = 32   # tokens that share a scale


class AXSKVCacheUnified(NamedTuple):
    """The cache's tensors, contiguous, on one GPU.  Lengths belong to the caller,
    who passes them to each call."""

    k_codes: torch.Tensor    # (B, heads, blocks, 32, D) int8
    k_scales: torch.Tensor   # (B, heads, blocks) float32
    v_codes: torch.Tensor    # (B, heads, blocks, D, 32) int8
    v_scales: torch.Tensor   # (B, heads, blocks) float32
    k_tail: torch.Tensor     # (B, heads, 32, D): the partial block's raw keys
    v_tail: torch.Tensor     # and values

    @classmethod
    def empty(cls, batch: int, heads: int, head_dim: int, max_tokens: int, dtype: torch.dtype = torch.float32,
              device: torch.device | str = "cuda") -> "AXSKVCacheUnified":
        """A cache for up to ``max_tokens`` tokens (rounded up to whole blocks) of
        ``batch`` sequences.  ``dtype``: that of the keys, values and queries."""
        nb = -(-max_tokens // CACHE_BLOCK)

        def codes(*shape):
            return torch.zeros(batch, heads, nb, *shape, dtype=torch.int8, device=device)

        def scales():
            return torch.zeros(batch, heads, nb, dtype=torch.float32, device=device)

        def tail():
            return torch.zeros(batch, heads, CACHE_BLOCK, head_dim, dtype=dtype, device=device)

        return cls(codes(CACHE_BLOCK, head_dim), scales(), codes(head_dim, CACHE_BLOCK), scales(), tail(), tail())

    @property
    def max_tokens(self) -> int:
        return self.k_codes.shape[2] * CACHE_BLOCK


def axs_cache_append_unified(cache: AXSKVCacheUnified, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor) -> None:
    """``k`` and ``v`` (B, n, heads, D) become tokens ``starts[b]`` .. ``starts[b] + n - 1``
    of sequence b; tokens from there on are forgotten.  ``starts`` (B) int64 or int32
    is read on the device: tokens past the cache's end are dropped, and all of a
    sequence whose start lies outside it.  A start past its block's
    first token needs the call before to have ended inside the same block, there or
    later: the block's earlier tokens come from the tail, which holds those of the last,
    partial block alone.  To go back further, append again from the first token of the
    block that this leads to."""
    _lib.ext().kv_append(*cache, k, v, starts)


def axs_cache_read_unified(cache: AXSKVCacheUnified, first: torch.Tensor, count: int) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values that the cache stands for, tokens ``first[b]`` ..
    ``first[b] + count - 1``, as float32 (B, count, heads, D); 0 outside the cache."""
    return _lib.ext().kv_read(*cache, first, count)


def axs_cache_attention_unified(
    q: torch.Tensor,
    cache: AXSKVCacheUnified,
    lengths: torch.Tensor,
    scale: float | None = None,
) -> torch.Tensor:
    """Attention of ``q`` (B, Tq, Hq, D), the last Tq of the ``lengths[b]`` tokens that the
    cache holds of sequence b, over them -> (B, Tq, Hq, D) of q's dtype.  Query t sees
    keys j <= lengths[b] - Tq + t (none: 0); Hq is a multiple of the cache's heads.
    ``lengths`` (B) int64 or int32 is read on the device.  ``scale`` is 1 / sqrt(D) if
    None, else any finite number.  No gradient."""
    return _lib.ext().kv_attention(q, *cache, lengths, scale)
