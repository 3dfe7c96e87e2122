"""The operators around the attention call in 64 bits, with a bound on what fp32 arithmetic and
one rounding may add, for their tests.

The bound of an output y: half a step of its type at y, plus `count` times 2^-24 of the sizes
that went into it.  `count` covers the longest chain of a row: a sum in order over a 64th of the
row and a tree over 64 partials (width / 64 + 6 additions, the fewest lanes that share a row of
more than 64 channels; at most 64 additions in order below that), the divisions and the root, and
up to 16 products and additions per element.
"""

from __future__ import annotations

import torch

STEP = 2.0 ** -24


def count(width: int) -> float:
    return max(64, width // 64 + 6) + 22


def half_step(y: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    info = torch.finfo(dtype)
    return (y.abs() * (info.eps / 2)).clamp_min(info.smallest_normal * info.eps / 2)


def norm(x, sizes, kind, weight, bias, eps, dims=(-1,)):
    """(norm of x over dims, sizes): x in 64 bits, and the error sizes of its elements."""
    if kind is None:
        return x, sizes
    mean = x.mean(dims, keepdim=True) if kind == "layer" else torch.zeros(())
    centred = x - mean.to(x)
    deviation = (centred.square().mean(dims, keepdim=True) + eps).sqrt()
    z = centred / deviation
    # A row's error moves every element through the mean, and each in proportion to itself
    # through the deviation (Cauchy-Schwarz: by no more than the root mean square error).
    spread = sizes.mean(dims, keepdim=True) + sizes.square().mean(dims, keepdim=True).sqrt()
    sizes = (sizes + mean.abs().to(x) + spread * (1 + z.abs())) / deviation + z.abs()
    if weight is not None:
        z, sizes = z * weight.double(), sizes * weight.double().abs()
    if bias is not None:
        z, sizes = z + bias.double(), sizes + bias.double().abs()
    return z, sizes


def rows(v, x):
    """A gate, scale or shift against [batch, tokens, width]."""
    v = v.double()
    return v[:, None] if v.ndim == 2 else v


def residual(x, branch=None, gate=None, scale=None, shift=None, *, kind=None, weight=None,
             bias=None, post=None, branch_weight=None, branch_bias=None, eps=1e-6):
    """((r, its bound), (y, its bound)) without their roundings: y None without a norm."""
    c = count(x.shape[-1]) * STEP
    r = x.double()
    sizes = r.abs()
    if branch is not None:
        f = branch.double()
        f, f_sizes = norm(f, f.abs(), post, branch_weight, branch_bias, eps)
        if gate is not None:
            f, f_sizes = f * rows(gate, x), f_sizes * rows(gate, x).abs()
        r, sizes = r + f, sizes + f_sizes
    first = (r, c * sizes)
    if kind is None:
        return first, None
    y, sizes = norm(r, sizes, kind, weight, bias, eps)
    if scale is not None:
        y, sizes = y * (1 + rows(scale, x)), sizes * (1 + rows(scale, x).abs())
    if shift is not None:
        y, sizes = y + rows(shift, x), sizes + rows(shift, x).abs()
    return first, (y, c * sizes)


def qk(x, axes, *, offset=0, pairing="interleaved", kind=None, weight=None, bias=None, eps=1e-6):
    """(rotated x, bound without its rounding) of [batch, heads, tokens, d]."""
    b, h, n, d = x.shape
    z = x.double()
    extent = d
    if kind == "rms_all":
        extent = h * d
        spread = lambda w: None if w is None else w.double().view(h, 1, d)  # noqa: E731
        z, sizes = norm(z, z.abs(), "rms", spread(weight), spread(bias), eps, dims=(1, 3))
    else:
        z, sizes = norm(z, z.abs(), kind, weight, bias, eps)
    if axes is not None:
        t, y, w = (a.shape[0] for a in axes)
        turns = torch.cat([
            axes[0].double()[:, None, None].expand(t, y, w, -1, 2),
            axes[1].double()[None, :, None].expand(t, y, w, -1, 2),
            axes[2].double()[None, None, :].expand(t, y, w, -1, 2)], dim=3).reshape(-1, d // 2, 2)
        cos, sin = torch.ones(n, d // 2).to(z), torch.zeros(n, d // 2).to(z)
        cos[offset:offset + t * y * w], sin[offset:offset + t * y * w] = turns.unbind(-1)
        part = (lambda v, i: v[..., i::2]) if pairing == "interleaved" else \
            (lambda v, i: v[..., i * (d // 2):(i + 1) * (d // 2)])
        out, grown = torch.empty_like(z), torch.empty_like(z)
        part(out, 0).copy_(part(z, 0) * cos - part(z, 1) * sin)
        part(out, 1).copy_(part(z, 1) * cos + part(z, 0) * sin)
        part(grown, 0).copy_(part(sizes, 0) * cos.abs() + part(sizes, 1) * sin.abs())
        part(grown, 1).copy_(part(sizes, 1) * cos.abs() + part(sizes, 0) * sin.abs())
        z, sizes = out, grown
    return z, count(extent) * STEP * sizes


def check(got: torch.Tensor, want, label: str) -> None:
    """Every element of `got` within half a step of its type and the arithmetic's bound."""
    exact, bound = want
    assert got.shape == exact.shape, label
    # the bound moves the value that is rounded, and with it the size of the half step
    limit = bound + half_step(exact.abs() + bound, got.dtype)
    off = (got.double() - exact).abs()
    assert torch.isfinite(got).all(), label
    worst = (off / limit).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{label}: off by {worst:.3f} of the bound"
