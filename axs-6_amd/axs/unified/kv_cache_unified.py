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


def axs_cache_shared_attention_unified(
    q: torch.Tensor,
    prefix: AXSKVCacheUnified,
    prefix_lengths: torch.Tensor,
    cache: AXSKVCacheUnified,
    lengths: torch.Tensor,
    scale: float | None = None,
) -> torch.Tensor:
    """Attention of sequences that share a prefix, whose codes are read once for all of them:
    of the B sequences of ``q`` (B, Tq, Hq, D), B a multiple of the P that ``prefix`` holds, number
    b continues prefix ``b // (B / P)``.  Its tokens are the ``prefix_lengths[b // (B / P)]`` of that
    prefix and then the ``lengths[b]`` of its own that ``cache`` holds, and ``q`` its last Tq:
    query t sees the keys at places j <= prefix + own - Tq + t of them (none: 0).
    -> (B, Tq, Hq, D) of q's dtype, that of both caches' tails.  ``prefix_lengths`` (P) and
    ``lengths`` (B), int64 or int32, are read on the device.  ``scale`` as in
    :func:`axs_cache_attention_unified`.  No gradient: a ``q`` that records one, or carries a
    forward-mode tangent, raises."""
    return _lib.ext().kv_shared_attention(q, *prefix, prefix_lengths, *cache, lengths, scale)


def axs_cache_copy_unified(
    cache: AXSKVCacheUnified,
    sources: torch.Tensor,
    lengths: torch.Tensor,
    target: AXSKVCacheUnified | None = None,
) -> None:
    """Sequence i of ``target`` becomes sequence ``sources[i]`` of ``cache``; ``target`` None:
    of the cache itself, in place, whatever the order of the sources.

    ``sources`` (target's sequences), or (G, n) for G groups: then its numbers count within the
    group's sequences of the cache, as the parents of :func:`axs_beam_select_unified` do.  One that
    is none of them (-1, say) leaves its sequence as it was.  ``lengths`` (cache's sequences):
    the tokens that each holds; whole blocks are copied and the raw rows of the partial one, and what
    lies behind them is left as it was.  Tokens past the end of either cache are dropped.  Both are int64
    or int32 and read on the device.  A target of its own has the cache's heads and dtype and
    shares no memory with it; its number of sequences and its capacity are its own.

    Reorder beams: ``sources=parents``.  Fork a prompt: one source for several sequences.  Close
    up a batch: the live sequences' numbers, then -1.  In place a group has up to 4096 sequences."""
    _lib.ext().kv_copy(*cache, sources, lengths, *(cache if target is None else target))
