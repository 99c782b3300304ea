"""``TypeCrossEntropy``: a classifier of node types and its loss in one."""
from __future__ import annotations

import torch
from torch import Tensor, nn

from .functional.type_loss import type_cross_entropy


class TypeCrossEntropy(nn.Module):
    """Cross entropy of ``types`` types by a learned table ``weight`` (types, channels), without keeping the logits (see
    :func:`~equitorch_b200.nn.functional.type_cross_entropy`).  The table starts from a normal distribution of variance one over the channels.  With that of a
    ``TypeEmbedding`` of one component call the function, on ``embedding.weight[:, 0]``."""

    def __init__(self, types: int, channels: int, reduction: str = "mean"):
        super().__init__()
        self.reduction = reduction
        self.weight = nn.Parameter(torch.empty(types, channels))
        self.reset_parameters()

    def reset_parameters(self) -> None:
        nn.init.normal_(self.weight, std=self.weight.shape[1] ** -0.5)

    def forward(self, x: Tensor, target: Tensor) -> Tensor:
        return type_cross_entropy(x, self.weight, target, self.reduction)

    def extra_repr(self) -> str:
        return f"{self.weight.shape[0]}, {self.weight.shape[1]}, reduction={self.reduction}"
