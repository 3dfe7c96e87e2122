"""Products of fp4 rows whose sums fp32 holds exactly, for their tests: with operands on the format's
grid and scales in a few binades, every product and every partial sum, in any order, is a multiple of
one unit and stays below 2^24 units.  Whatever order the sum is taken in, it has no rounding, and the
result is the 64-bit sum's bit for bit; a block left out, a sum kept in 16 bits or a sum rounded
beside a large bias is not."""

from __future__ import annotations

import torch

POWERS = 3              # of two among the scales
UNIT = 0.25             # the product of the smallest codes at the smallest scales


def operand(g: torch.Generator, rows: int, width: int) -> torch.Tensor:
    """fp32 rows that are their own fp4 form: each block of 32 values holds a 6, the largest code, so
    that its scale is the power of two that it was made with."""
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6])
    blocks = -(-width // 32)
    index = torch.randint(0, 8, (rows, blocks * 32), generator=g)
    index[:, ::32] = 7
    sign = 1 - 2 * torch.randint(0, 2, index.shape, generator=g)
    power = torch.randint(0, POWERS, (rows, blocks), generator=g).repeat_interleave(32, 1)
    return (grid[index] * sign * 2 ** power)[:, :width].contiguous()


def check_exact(got: torch.Tensor, x: torch.Tensor, w: torch.Tensor, bias, label: str) -> None:
    """got against the sum of 64-bit operands, rounded to fp32 (it is no rounding without a bias) and
    then to got's type."""
    size = x.double().abs() @ w.double().abs().T
    assert size.max() < 2.0 ** 24 * UNIT, "the operands' sums may need more than 24 bits"
    want = x.double() @ w.double().T
    if bias is not None:
        want = want + bias.double()
    want = want.float().to(got.dtype)
    assert got.shape == want.shape, label
    off = got != want
    assert not off.any(), f"{label}: {int(off.sum())} of {got.numel()} differ"
