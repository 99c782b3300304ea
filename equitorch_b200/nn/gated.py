"""``GatedLinear``: two projections, the activation of one and their product."""
from __future__ import annotations

import torch
from torch import Tensor, nn

from ..ops.gated_op import ACTIVATIONS
from .functional.gated import gated_linear
from .init import initialize_linear


class GatedLinear(nn.Module):
    """``act(x W[0]) * (x W[1])`` on invariant features ``(..., channels_in)`` -> ``(..., hidden)``, the first half of a gated
    feed-forward block (an :class:`IrrepWiseLinear` or any linear layer is the second).  ``weight`` is ``(2, channels_in, hidden)``,
    initialised as the other linear layers are."""

    def __init__(self, channels_in: int, hidden: int, activation: str = "silu"):
        super().__init__()
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation should be in {list(ACTIVATIONS)}, got {activation}")
        self.channels_in, self.hidden, self.activation = channels_in, hidden, activation
        self.weight = nn.Parameter(torch.empty(2, channels_in, hidden))
        initialize_linear(self.weight)

    def forward(self, input: Tensor) -> Tensor:
        return gated_linear(input, self.weight, self.activation)

    def extra_repr(self) -> str:
        return f"{self.channels_in}, {self.hidden}, activation={self.activation}"
