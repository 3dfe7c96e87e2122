"""The attention half of a video transformer block around ``Operator.attend``.

What the reference's processors and the blocks around them do with torch modules
(recap/models/hunyuan.py:79-154): the modulated norm of the residual stream, the projections,
the queries' and keys' norm and rotation, the attention call, the output projection, and the
gated residual with the next half's modulated norm.  The projections are the model's own
modules, or ``MicroscaledLinear``s in 4 bits; everything between them runs on the HIP kernels.  A
model integration builds one per layer in its ``build_operator`` and calls it in the block's forward.

It is a block of one stream: one set of projections, norms and modulations for the tokens of the
whole sequence.  A block whose text tokens have their own calls the kernels itself, each stream's
queries and keys with ``q_out`` and ``k_out`` in its part of the joint sequence.
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Callable

import torch

from . import kernels as K
from .microscale import MicroscaledLinear
from .operator import Operator

Projection = Callable[[torch.Tensor], torch.Tensor]


@dataclass
class AttentionBlock:
    """One layer's attention half: called with the residual stream ``[B, N, width]`` and this
    step's modulation, it returns the stream after the attention and its normalised form for
    the next half."""

    operator: Operator
    layer: int
    heads: int
    to_q: Projection                        # [B, N, width] -> [B, N, heads * d]
    to_k: Projection
    to_v: Projection
    to_out: Projection                      # [B, N, heads * d] -> [B, N, width]
    axes: tuple[torch.Tensor, ...] | None = None   # rotary_axes of the layout's video grid
    pairing: str = "interleaved"
    qk_norm: str | None = None              # kernels.qk_rotary's norm, weights and biases
    q_weight: torch.Tensor | None = None
    k_weight: torch.Tensor | None = None
    q_bias: torch.Tensor | None = None
    k_bias: torch.Tensor | None = None
    norm: str = "layer"                     # before the attention
    weight: torch.Tensor | None = None
    bias: torch.Tensor | None = None
    branch_norm: str | None = None          # of the attention's output
    branch_weight: torch.Tensor | None = None
    branch_bias: torch.Tensor | None = None
    next_norm: str = "layer"                # before the next half
    next_weight: torch.Tensor | None = None
    next_bias: torch.Tensor | None = None
    eps: float = 1e-6                       # of the norm before the attention
    dtype: torch.dtype | None = None        # of the projections; None: the stream's
    qk_eps: float | None = None             # of the queries' and keys' norm; None: eps
    next_eps: float | None = None           # of the output's norm and the next half's; None: eps

    def __call__(self, x: torch.Tensor, scale: torch.Tensor | None = None,
                 shift: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                 next_scale: torch.Tensor | None = None,
                 next_shift: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """(x + gate * attention(norm(x) * (1 + scale) + shift), and the norm of that modulated by
        next_scale and next_shift)."""
        layout = self.operator.layout
        layout._check(x)
        if self.axes is not None:
            grid = [t.shape[0] for t in self.axes]
            if math.prod(grid) != layout.video_tokens:
                raise ValueError(f"the rotary axes span {grid}, the layout has "
                                 f"{layout.video_tokens} video tokens")
        y = K.norm_modulate(x, scale, shift, norm=self.norm, weight=self.weight, bias=self.bias,
                            eps=self.eps, dtype=self.dtype)
        projections = self.to_q, self.to_k, self.to_v
        if all(isinstance(p, MicroscaledLinear) for p in projections):
            rows = K.mx_quantise(y)     # once for the three
            parts = [p(rows, dtype=p.dtype or y.dtype) for p in projections]
        else:
            parts = [p(y) for p in projections]
        query, key, value = (t.unflatten(-1, (self.heads, -1)).transpose(1, 2) for t in parts)
        query, key = K.qk_rotary(query, key, self.axes, offset=layout.video_offset,
                                 pairing=self.pairing, norm=self.qk_norm,
                                 q_weight=self.q_weight, k_weight=self.k_weight,
                                 q_bias=self.q_bias, k_bias=self.k_bias,
                                 eps=self.eps if self.qk_eps is None else self.qk_eps)
        out = self.operator.attend(self.layer, query, key, value)
        branch = self.to_out(out.transpose(1, 2).flatten(2))
        return K.gated_residual_norm(
            x, branch, gate, next_scale, next_shift, norm=self.next_norm, weight=self.next_weight,
            bias=self.next_bias, branch_norm=self.branch_norm, branch_weight=self.branch_weight,
            branch_bias=self.branch_bias, eps=self.eps if self.next_eps is None else self.next_eps)
