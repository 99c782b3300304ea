"""``TypeEmbedding``: features by node or edge type."""
from __future__ import annotations

import torch
from torch import Tensor, nn

from .functional.embedding import type_embedding


class TypeEmbedding(nn.Module):
    """Learned features of ``num_types`` node or edge types: types ``(...)`` int64 -> ``(..., components, channels)`` in the layout
    of the other layers, ``scale`` times a row of ``weight`` (``num_types, components, channels``).  A type outside
    ``[0, num_types)`` gives zeros and no gradient.  Only invariant components keep the network equivariant, so
    ``components`` is the number of scalar irreps."""

    def __init__(self, num_types: int, channels: int, components: int = 1, scale: float = 1.0):
        super().__init__()
        self.num_types, self.channels, self.components, self.scale = num_types, channels, components, float(scale)
        self.weight = nn.Parameter(torch.empty(num_types, components, channels))
        nn.init.normal_(self.weight)

    def forward(self, types: Tensor) -> Tensor:
        return type_embedding(types, self.weight, self.scale)

    def extra_repr(self) -> str:
        return f"{self.num_types}, {self.channels}, components={self.components}, scale={self.scale}"
