"""Rotary positions of queries and keys (the reference's attention has learned
positions only; this operator is this library's).

``rotary_table`` builds the cosines and sines once, in float64;
``axs_rotary_unified`` rotates queries and keys by them in one launch, with
gradients, in either layout and for any even part of the head.
"""
from __future__ import annotations

import math

import torch

from axs import _lib


def rotary_table(
    rotary_dim: int,
    max_positions: int,
    base: float = 10000.0,
    scaling: str | None = None,
    factor: float = 1.0,
    original_positions: int | None = None,
    device: torch.device | str | None = None,
) -> torch.Tensor:
    """The (max_positions, rotary_dim) float32 table that :func:`axs_rotary_unified`
    reads: row p holds cos(p w_i), then sin(p w_i), for the rotary_dim / 2
    frequencies w_i = base ** (-2 i / rotary_dim).

    ``scaling`` stretches a model trained on ``original_positions`` to ``factor``
    times as many:

    * ``"linear"`` -- every w_i divided by factor (positions interpolated);
    * ``"base"`` -- base times factor ** (d / (d - 2)): the lowest frequency is
      divided by factor, the highest stays;
    * ``"parts"`` -- by wavelength: frequencies that turn 32 times or more within
      original_positions stay, those that turn at most once are divided by
      factor, a linear ramp over i between; the table is multiplied by
      0.1 ln(factor) + 1, which sharpens the longer softmax.
    """
    if rotary_dim < 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and not negative, got {rotary_dim}")
    if max_positions < 1:
        raise ValueError(f"max_positions must be positive, got {max_positions}")
    if not (base > 1.0 and factor >= 1.0):
        raise ValueError(f"base must be over 1 and factor at least 1, got {base} and {factor}")
    if scaling not in (None, "linear", "base", "parts"):
        raise ValueError(f"scaling must be None, 'linear', 'base' or 'parts', got {scaling!r}")
    if scaling == "base" and rotary_dim > 2:
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    inv = base ** (-2.0 * i / max(rotary_dim, 1))
    gain = 1.0
    if scaling == "linear":
        inv = inv / factor
    elif scaling == "parts":
        if original_positions is None or original_positions < 1:
            raise ValueError("scaling 'parts' needs original_positions")

        def turns(n: float) -> float:   # the index whose frequency turns n times
            return rotary_dim * math.log(original_positions / (2 * math.pi * n)) / (2 * math.log(base))

        # high may lie past the last index: no frequency is then divided in full
        low, high = max(math.floor(turns(32.0)), 0), math.ceil(turns(1.0))
        ramp = torch.where(i >= high, 1.0, ((i - low) / max(high - low, 1)).clamp(0.0, 1.0))
        inv = inv / factor * ramp + inv * (1.0 - ramp)
        gain = 0.1 * math.log(factor) + 1.0
    angle = torch.arange(max_positions, dtype=torch.float64)[:, None] * inv
    return (torch.cat([angle.cos(), angle.sin()], 1) * gain).float().to(device or "cpu")


def axs_rotary_unified(
    q: torch.Tensor,
    k: torch.Tensor | None,
    table: torch.Tensor,
    positions: torch.Tensor | None = None,
    interleaved: bool = False,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """``q`` (B, T, Hq, D) and ``k`` (B, T, Hkv, D; or None) with their heads' first
    ``table.shape[1]`` values rotated by their positions: pairs (x[i], x[i + R/2]),
    or neighbours (x[2i], x[2i + 1]) with ``interleaved``; the rest is copied.

    ``positions``: int64 or int32, (T) or (B, T); None is 0..T-1.  They are read on
    the device: one outside the table gives NaN.  float32, bfloat16 or float16,
    computed in float32 and rounded once; contiguous results; gradients for q and k.
    """
    return _lib.ext().rotary(q, k, table, positions, interleaved)
