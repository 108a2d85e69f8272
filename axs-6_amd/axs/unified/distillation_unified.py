"""Distillation from a teacher's top logits: the loss that trains a quantized
model towards its full-precision original (the reference has none).
"""
from __future__ import annotations

from typing import Literal

import torch

from axs import _lib

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def axs_distillation_loss_unified(
    student_logits: torch.Tensor,
    teacher_values: torch.Tensor,
    teacher_indices: torch.Tensor,
    temperature: float = 1.0,
    weights: torch.Tensor | None = None,
    reduction: Literal["mean", "sum", "none"] = "mean",
) -> torch.Tensor:
    """T^2 KL(p || q) of each row, p = softmax(teacher_values / T) over the teacher's
    top entries and q = softmax(student_logits / T) over all classes.

    ``student_logits`` (*, V) float32, bfloat16 or float16; ``teacher_values`` (*, K)
    floats and ``teacher_indices`` (*, K) int64 or int32, each entry's class: one below
    0 is left out, one at or past V makes its row NaN; ``weights`` (*) per row, a row of
    weight 0 is not read.  ``"mean"`` is the weighted mean (0 where the weights sum to
    0), ``"sum"`` the weighted sum, ``"none"`` the weighted rows.  float32 result; the
    gradient T w (q - p), for the student's logits alone, is rounded once to their type;
    its time grows with K^2, since classes may repeat: K is meant to be some hundreds.
    """
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be 'mean', 'sum' or 'none', got {reduction!r}")
    return _lib.ext().distill(student_logits, teacher_values, teacher_indices, temperature, weights,
                              _REDUCTIONS[reduction])
