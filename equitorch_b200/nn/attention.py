"""``GraphAttention``: attention within the graphs of a packed batch."""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor, nn

from ..graph import PackedGraphs
from .functional.attention import graph_attention


class GraphAttention(nn.Module):
    """Attention of ``num_heads`` heads among the nodes of each graph (see :func:`~equitorch_b200.nn.functional.graph_attention`):
    q, k, v ``(N, components, channels)``, a :class:`~equitorch_b200.graph.PackedGraphs` and, with ``distance_bias``, positions
    ``(N, 3)``.  The slopes of the distance term are learned, ``slope`` (num_heads,), float32, starting from 2^(-8 h / num_heads) for
    h = 1 .. num_heads; a module moved to another type computes with them in float32."""

    def __init__(self, num_heads: int, distance_bias: bool = True, cap: Optional[float] = None, scale: Optional[float] = None):
        super().__init__()
        self.num_heads, self.cap, self.scale = num_heads, cap, scale
        self.slope = nn.Parameter(2.0 ** (-8.0 * torch.arange(1, num_heads + 1) / num_heads)) if distance_bias else None

    def forward(self, q: Tensor, k: Tensor, v: Tensor, graphs: PackedGraphs, pos: Optional[Tensor] = None) -> Tensor:
        if (pos is None) != (self.slope is None):
            raise ValueError("positions are needed with distance_bias and not taken without")
        slope = None if self.slope is None else self.slope.float()
        return graph_attention(q, k, v, graphs, self.num_heads, self.scale, self.cap, pos, slope)

    def extra_repr(self) -> str:
        return f"{self.num_heads}, distance_bias={self.slope is not None}, cap={self.cap}, scale={self.scale}"
