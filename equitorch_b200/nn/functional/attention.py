"""Attention within the graphs of a packed batch."""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from ...graph import PackedGraphs
from ...ops import attention_op as _ops


class _GraphAttention(Function):
    @staticmethod
    def forward(ctx, q, k, v, pos, slope, graphs, heads, scale, cap):
        out, stats = _ops.attention_forward(q, k, v, graphs, heads, scale, cap, pos, slope, any(ctx.needs_input_grad))
        ctx.save_for_backward(q, k, v, pos, slope, out, stats)
        ctx.graphs, ctx.heads, ctx.scale, ctx.cap = graphs, heads, scale, cap
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        q, k, v, pos, slope, out, stats = ctx.saved_tensors
        need = ctx.needs_input_grad
        dq, dk, dv, dslope, dpos = _ops.attention_backward(grad, q, k, v, ctx.graphs, ctx.heads, ctx.scale, ctx.cap, pos, slope, out, stats,
                                                           need[3] or need[4])
        return (dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, dpos if need[3] else None,
                dslope if need[4] else None, None, None, None, None)


def graph_attention(q: Tensor, k: Tensor, v: Tensor, graphs: PackedGraphs, num_heads: int, scale: Optional[float] = None,
                    cap: Optional[float] = None, pos: Optional[Tensor] = None, slope: Optional[Tensor] = None) -> Tensor:
    r"""Every node attends to the nodes of its own graph, itself among them:

    .. math:: out_i = \sum_j softmax_j(s_{ij}) v_j, \quad s_{ij} = cap \tanh(scale \langle q_i, k_j \rangle / cap) - slope_h |p_i - p_j|

    ``q``, ``k``, ``v`` are ``(N, components, channels)``, float32 or bfloat16, of any strides (three times as fast where each component's
    channels of a head are whole 16 bytes on 16-byte boundaries); the channels are split over
    ``num_heads`` heads of at most 128 values (components times channels a head) a node.  A head's inner product runs over all
    components of its channels, so with features of one sequence of irreps in the basis of this package the scores do not change
    under rotations and the result turns as the features do.

    ``scale``: one over the root of a head's values where not given.  ``cap`` (1e-12 to 1e12): the products, not the distances, are capped;
    without it they are taken as they are.  ``pos`` (N, 3) and ``slope`` (num_heads,), float32, come together; without them there is no
    distance term.  Nodes of no graph get zeros, and graphs do not touch each other, whatever values they hold.

    Differentiable once in ``q``, ``k``, ``v``, ``pos`` and ``slope``: forces from ``pos`` at inference, but no training on forces through it.
    The gradient of a distance is zero where two nodes coincide; nodes closer than 1e-15 count as closer than they are.  Sums in float32, one
    order of sums, no atomics; of bfloat16 features, weights and their gradients are rounded to bfloat16 for the products."""
    _ops.check(q, k, v, graphs, num_heads, scale, cap, pos, slope)
    if scale is None:
        scale = (q.shape[1] * q.shape[2] // num_heads) ** -0.5
    return _GraphAttention.apply(q, k, v, pos, slope, graphs, num_heads, float(scale), None if cap is None else float(cap))
