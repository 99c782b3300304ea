"""``AddRMSNorm``: root-mean-square norm with the residual's addition before it."""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor, nn

from .functional.residual_norm import add_rms_norm


class AddRMSNorm(nn.Module):
    """The norm of :func:`~equitorch_b200.nn.functional.add_rms_norm` with a learned weight for each channel (ones at first; none without
    ``affine``): features and the residual ``(N, components, channels)`` or ``(N, channels)`` to the normalised sum and the sum."""

    def __init__(self, channels: int, eps: float = 1e-6, affine: bool = True):
        super().__init__()
        self.channels, self.eps = channels, eps
        self.weight = nn.Parameter(torch.ones(channels)) if affine else None

    def reset_parameters(self) -> None:
        if self.weight is not None:
            nn.init.ones_(self.weight)

    def forward(self, x: Tensor, residual: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
        if x.shape[-1] != self.channels:
            raise ValueError(f"{self.channels} channels expected, got {tuple(x.shape)}")
        return add_rms_norm(x, residual, self.weight, self.eps)

    def extra_repr(self) -> str:
        return f"{self.channels}, eps={self.eps}, affine={self.weight is not None}"
