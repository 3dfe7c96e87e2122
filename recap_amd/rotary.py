"""Rotary tables of a video's (time, height, width) axes for ``kernels.qk_rotary``.

A head's d / 2 frequencies are shared out over the axes; an axis with ``c`` channels has the
frequencies ``theta ** (-2 i / c)``, and a token turns by its own coordinate on each axis.  The
tables hold one row per coordinate of an axis instead of one per token (103 rows instead of
32,760 for a grid of 21 x 30 x 52), so they stay in the caches while Q and K stream past.
"""

from __future__ import annotations

from typing import Sequence

import torch


def rotary_axes(grid: Sequence[int], channels: Sequence[int], *, theta: float = 10000.0,
                positions: Sequence | None = None, device=None) -> tuple[torch.Tensor, ...]:
    """(cos, sin) tables, fp32 ``[length, channels / 2, 2]``, of the axes (time, height, width).

    ``grid`` is (T, H, W), ``channels`` how many of a head's channels each axis turns (even; 0
    leaves an axis out).  ``positions`` gives an axis other coordinates than 0, 1, ...: three
    sequences of the axes' lengths (fractions for a resized grid), or None for an axis.
    Angles, sines and cosines are taken in 64 bits and rounded once."""
    grid, channels = [int(n) for n in grid], [int(c) for c in channels]
    if len(grid) != 3 or len(channels) != 3 or min(grid) < 1:
        raise ValueError(f"grid {grid} and channels {channels} must be (time, height, width)")
    if min(channels) < 0 or any(c % 2 for c in channels):
        raise ValueError(f"channels {channels} must be even")
    if not theta > 0:
        raise ValueError(f"theta must be positive, got {theta}")
    positions = [None] * 3 if positions is None else list(positions)
    if len(positions) != 3:
        raise ValueError("positions must have one entry per axis")
    tables = []
    for length, count, where in zip(grid, channels, positions):
        at = torch.arange(length, dtype=torch.float64) if where is None else \
            torch.as_tensor(where, dtype=torch.float64, device="cpu")
        if tuple(at.shape) != (length,):
            raise ValueError(f"positions of shape {tuple(at.shape)} for an axis of {length}")
        turn = float(theta) ** (-torch.arange(0, count, 2, dtype=torch.float64) / max(count, 1))
        angle = at[:, None] * turn
        tables.append(torch.stack((angle.cos(), angle.sin()), dim=-1).to(torch.float32).to(device))
    return tuple(tables)
