"""Projections with 4-bit weights and activations, over ``kernels.mx_linear``."""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import kernels as K
from .kernels import Microscaled


@dataclass(frozen=True)
class MicroscaledLinear:
    """A linear layer whose weight ``[outputs, width]`` is kept in fp4 and whose input is brought into
    fp4 on its way in, for inference: called with rows ``[..., width]`` (or with a Microscaled, rows
    that several layers share), it returns ``[..., outputs]`` of ``dtype`` (None: the input's; bfloat16
    for codes).  ``AttentionBlock`` takes it in a projection's place."""

    weight: Microscaled
    bias: torch.Tensor | None = None
    dtype: torch.dtype | None = None

    @classmethod
    @torch.no_grad()
    def from_linear(cls, linear: torch.nn.Linear, dtype: torch.dtype | None = None) -> "MicroscaledLinear":
        """From a torch layer on the GPU, as it is now: later changes to it are not seen."""
        bias = None if linear.bias is None else linear.bias.detach().clone()
        return cls(K.mx_quantise(linear.weight.detach()), bias, dtype)

    def __call__(self, x: torch.Tensor | Microscaled, *,
                 dtype: torch.dtype | None = None) -> torch.Tensor:
        return K.mx_linear(x, self.weight, self.bias, dtype=dtype or self.dtype)
