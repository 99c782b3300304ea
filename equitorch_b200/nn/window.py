"""``WindowAttention``: attention within a window along the chains of a packed batch."""
from __future__ import annotations

from typing import Optional

from torch import Tensor, nn

from ..graph import PackedGraphs
from .functional.window import window_attention


class WindowAttention(nn.Module):
    """Attention of ``num_heads`` heads of queries to the nodes near each along its chain and to the chain's first ones (see
    :func:`~equitorch_b200.nn.functional.window_attention`): q ``(N, components, channels)``, k and v of ``kv_heads`` heads and a
    :class:`~equitorch_b200.graph.PackedGraphs`."""

    def __init__(self, num_heads: int, before: int, after: int = 0, sinks: int = 0, kv_heads: Optional[int] = None, scale: Optional[float] = None):
        super().__init__()
        self.num_heads, self.before, self.after, self.sinks, self.kv_heads, self.scale = num_heads, before, after, sinks, kv_heads, scale

    def forward(self, q: Tensor, k: Tensor, v: Tensor, graphs: PackedGraphs) -> Tensor:
        return window_attention(q, k, v, graphs, self.num_heads, self.before, self.after, self.sinks, self.kv_heads, self.scale)

    def extra_repr(self) -> str:
        return f"{self.num_heads}, before={self.before}, after={self.after}, sinks={self.sinks}, kv_heads={self.kv_heads}, scale={self.scale}"
