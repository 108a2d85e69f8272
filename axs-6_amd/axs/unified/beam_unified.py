"""Beam search: the choice of the best continuations over beams and vocabulary.

``axs_beam_select_unified`` scores every continuation of every beam and keeps the best,
from one reading of the logits.  The reference has no counterpart.
"""
from __future__ import annotations

import torch

from axs import _lib


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
    (at most 1024) of G sequences, and ``scores`` (G, W) float32, the beams' log probabilities.
    Token j after beam w scores ``scores[w] + log_softmax(logits[w])[j]``; equal ones stand
    in the order of beam, then token.  ``finished`` (G, W) bool: a beam that has ended goes
    on as one candidate, the token ``end`` with the beam's own score; its logits are not read.

    A logit of -inf is no candidate, and a beam of score -inf has none (start a search from one
    prompt with scores 0, -inf, -inf, ...).  Slots for which no candidate is left have the score
    -inf, parent 0 and token 0.  A NaN or +inf in a logit or score that counts makes the
    sequence's scores NaN, its parents and tokens 0.

    Sums and comparisons are in float64, the scores are rounded once.  No gradient."""
    return _lib.ext().beam_select(logits, scores, finished, end, count)
