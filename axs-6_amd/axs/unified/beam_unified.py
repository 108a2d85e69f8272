"""Beam search: the choice of the best continuations over beams and vocabulary.

``axs_beam_select_unified`` scores every continuation of every beam and keeps the best,
from one reading of the logits; ``axs_beam_search_unified`` is the loop around it that
keeps the 8-bit caches in step with the beams.  The reference has no counterpart.
"""
from __future__ import annotations

from collections.abc import Callable, Sequence

import torch

from axs import _lib
from axs.unified.kv_cache_unified import AXSKVCacheUnified, axs_cache_copy_unified


def axs_beam_select_unified(
    logits: torch.Tensor,
    scores: torch.Tensor,
    finished: torch.Tensor | None = None,
    end: int | None = None,
    count: int | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The ``count`` (None: as many as beams; at most 128) best continuations of each sequence's
    beams: (scores float32, parents int64, tokens int64), each (G, count), best first.

    ``logits`` (G, W, V) float32, bfloat16 or float16, those of the next token after each of W beams
    (at most 1024, and 65535 of all sequences) of G sequences, and ``scores`` (G, W) float32, the beams' log probabilities.
    Token j after beam w scores ``scores[w] + log_softmax(logits[w])[j]``; equal ones stand
    in the order of beam, then token.  ``finished`` (G, W) bool: a beam that has ended goes
    on as one candidate, the token ``end`` with the beam's own score; its logits are not read.

    A logit of -inf is no candidate, and a beam of score -inf has none (start a search from one
    prompt with scores 0, -inf, -inf, ...).  Slots for which no candidate is left have the score
    -inf, parent 0 and token 0.  A NaN or +inf in a logit or score that counts makes the
    sequence's scores NaN, its parents and tokens 0.

    Exponentials are float32, each off by some 2^-24 of itself; their sums, the scores and comparisons
    are float64, and the scores are rounded once.  No gradient: logits or scores that record one, or
    carry a forward-mode tangent, raise."""
    return _lib.ext().beam_select(logits, scores, finished, end, count)


@torch.no_grad()
def axs_beam_search_unified(
    step: Callable[[torch.Tensor, torch.Tensor], torch.Tensor],
    logits: torch.Tensor,
    caches: Sequence[AXSKVCacheUnified],
    beams: int,
    steps: int,
    end: int | None = None,
    starts: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """The ``beams`` (at most 128) best continuations by ``steps`` tokens of each of G prompts:
    (scores (G, beams) float32, log probabilities; tokens (G, beams, steps) int64), best first.

    ``logits`` (G, V), those of the token after each prompt.  ``caches``, one a layer, hold the
    G * beams sequences of the beams: their own tokens alone where the prompt is a shared prefix,
    else the prompts forked (:func:`axs_cache_copy_unified`) and ``starts`` (G * beams), the tokens
    that each holds (None: 0).  ``step(tokens (G * beams, 1), starts (G * beams))`` appends those
    tokens to the caches and returns the logits of the next, (G * beams, V) or (G * beams, 1, V);
    it is called ``steps - 1`` times.  A beam that chose ``end`` goes on as it, at its score.
    Slots for which there is no candidate have the score -inf.  At the end the caches' sequences
    are those of the returned beams, without their last tokens: ``steps - 1`` more each."""
    if beams < 1 or steps < 1:
        raise ValueError(f"{beams} beams of {steps} steps")
    G = logits.shape[0]
    scores, parents, tokens = axs_beam_select_unified(
        logits[:, None], torch.zeros(G, 1, dtype=torch.float32, device=logits.device), count=beams)
    if starts is None:
        starts = torch.zeros(G * beams, dtype=torch.int64, device=logits.device)
    out = tokens[..., None]
    finished = None if end is None else tokens == end
    for i in range(1, steps):
        logits = step(tokens.view(-1, 1), starts)
        starts = starts + 1
        scores, parents, tokens = axs_beam_select_unified(
            logits.reshape(G, beams, logits.shape[-1]), scores, finished, end)
        out = torch.cat([out.gather(1, parents[..., None].expand(-1, -1, i)), tokens[..., None]], -1)
        if end is not None:
            finished = finished.gather(1, parents) | (tokens == end)
        for cache in caches:
            axs_cache_copy_unified(cache, parents, starts)
        starts = starts.view(G, beams).gather(1, parents).flatten()
    return scores, out
