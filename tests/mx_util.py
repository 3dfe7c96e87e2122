"""Microscaled rows and their product in 64 bits, for their tests."""

from __future__ import annotations

import torch

BLOCK = 32
FILL = {"fp4": 256, "int8": 32}
GRID = {"fp4": [0, 0.5, 1, 1.5, 2, 3, 4, 6], "int8": [c / 64 for c in range(128)]}
# A block's scale is the smallest power of two with which its largest magnitude stays under this.
LIMIT = {"fp4": 7.0, "int8": 127.5 / 64}


def filled(width: int, format: str) -> int:
    return -(-width // FILL[format]) * FILL[format]


def quantise(x: torch.Tensor, format: str):
    """(index of each value's magnitude [..., filled] with the sign apart, scale bytes): on the CPU,
    in 64 bits, each value compared with the middles between the codes."""
    x = x.detach().cpu().double()
    v = torch.zeros(*x.shape[:-1], filled(x.shape[-1], format), dtype=torch.float64)
    v[..., :x.shape[-1]] = x
    v = v.unflatten(-1, (-1, BLOCK))
    bad = ~torch.isfinite(v).all(-1, keepdim=True)
    v = torch.where(bad, 0.0, v)
    top = v.abs().amax(-1, keepdim=True)
    scale = torch.full_like(top, -127.0)
    for e in range(-127, 128):
        scale = torch.where(top >= LIMIT[format] * 2.0 ** e, float(e + 1), scale)
    scale = scale.clamp(max=127 if format == "int8" else 126)
    grid = torch.tensor(GRID[format], dtype=torch.float64)
    middles = (grid[1:] + grid[:-1]) / 2
    size = (v * 2.0 ** -scale).abs()
    low, high = torch.bucketize(size, middles), torch.bucketize(size, middles, right=True)
    index = torch.where(low % 2 == 0, low, high)
    byte = torch.where(bad, 255.0, scale + 127).squeeze(-1).to(torch.uint8)
    return index.flatten(-2), torch.signbit(v).flatten(-2), byte


def pack(index, negative, format: str) -> torch.Tensor:
    """Codes as they lie in memory."""
    if format == "int8":
        return torch.where(negative, -index, index).to(torch.int8)
    code = (index + 8 * negative).to(torch.uint8)
    return code[..., ::2] | code[..., 1::2] << 4


def unpack(codes: torch.Tensor, format: str):
    """(index, negative) of codes."""
    codes = codes.cpu()
    if format == "int8":
        return codes.long().abs(), codes < 0
    pairs = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).long()
    return pairs & 7, pairs >= 8


def values(index, negative, byte, format: str, width: int) -> torch.Tensor:
    """The 64-bit values [..., width] they stand for."""
    v = torch.tensor(GRID[format], dtype=torch.float64)[index]
    v = torch.where(negative, -v, v).unflatten(-1, (-1, BLOCK))
    byte = byte.cpu()
    v = v * 2.0 ** (byte.double() - 127)[..., None]
    v = torch.where((byte == 255)[..., None], float("nan"), v)
    return v.flatten(-2)[..., :width]


def read(m) -> torch.Tensor:
    return values(*unpack(m.codes, m.format), m.scales, m.format, m.width)


def rounded(x: torch.Tensor, format: str) -> torch.Tensor:
    index, negative, byte = quantise(x, format)
    return values(index, negative, byte, format, x.shape[-1])


def check_product(got, x, w, bias, label: str) -> None:
    """got against x @ w.T + bias of 64-bit values.  Bound: half a step of its type, and 2^-23 (one
    step, so that an addition may also cut off) for each of width + 1 additions in turn, of the sum
    of the magnitudes."""
    want, size = x @ w.T, x.abs() @ w.abs().T
    if bias is not None:
        bias = bias.to(want.device).double()
        want, size = want + bias, size + bias.abs()
    limit = (x.shape[-1] + 1) * 2.0 ** -23 * size
    info = torch.finfo(got.dtype)
    limit = limit + ((want.abs() + limit) * (info.eps / 2)).clamp_min(info.smallest_normal * info.eps / 2)
    assert got.shape == want.shape, label
    got = got.to(want.device).double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{label}: NaN"
    ok = ~torch.isnan(want)
    off = ((got - want).abs() / limit)[ok]
    worst = off.max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{label}: off by {worst:.3f} of the bound"
