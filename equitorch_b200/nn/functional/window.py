"""Attention within a window along the chains of a packed batch, and for one new node of every chain."""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from ...graph import PackedGraphs
from ...ops import window_op as _ops


class _WindowAttention(Function):
    @staticmethod
    def forward(ctx, q, k, v, graphs, heads, kv_heads, window, scale):
        out, rest, stats = _ops.window_forward(q, k, v, graphs, heads, kv_heads, window, scale, any(ctx.needs_input_grad))
        ctx.save_for_backward(q, k, v, out, rest, stats)
        ctx.args = graphs, heads, kv_heads, window, scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        q, k, v, out, rest, stats = ctx.saved_tensors
        grads = _ops.window_backward(grad, q, k, v, *ctx.args, out, rest, stats)
        return (*(g if need else None for g, need in zip(grads, ctx.needs_input_grad)), *[None] * 5)


def window_attention(q: Tensor, k: Tensor, v: Tensor, graphs: PackedGraphs, num_heads: int, before: int, after: int = 0, sinks: int = 0,
                     kv_heads: Optional[int] = None, scale: Optional[float] = None) -> Tensor:
    r"""Every node attends to the nodes near it along its chain and to the chain's first ones:

    .. math:: out_i = \sum_j softmax_j(scale \langle q_i, k_j \rangle) v_j, \quad j \le i + after, \quad j \ge i - before \text{ or } j < sinks

    with nodes counted from the start of their chain, a graph of ``graphs`` whose nodes are in order.  ``after = 0`` reads chains in their order (and
    a node sees no first node that is still ahead of it); the first ``sinks`` nodes are for tokens that all others are to see, or for
    what the softmax does not need elsewhere.

    ``q`` is ``(N, components, channels)`` of ``num_heads`` heads, ``k`` and ``v`` of ``kv_heads`` (as many where not given, else a divisor: head h has
    the keys of head ``h // (num_heads // kv_heads)``); float32 or bfloat16, of any strides, at most 128 values (components times channels a head) a
    head.  Inner products run over all components, as in :func:`graph_attention`, so equivariant features stay so.  ``scale``: one over the root
    of a head's values where not given.  Nodes of no graph get zeros.  What a node does not see does not reach it, not even a NaN, and chains do not
    touch each other; next to values that are not finite a row's sums may be of another order, and its weights not rounded.

    Differentiable once in ``q``, ``k`` and ``v``.  Sums in float32, one order of sums, no atomics; of bfloat16 features, weights and score
    gradients are rounded to bfloat16 for the products (of small batches, to two parts for the gradients of keys and values).  Beside its inputs and result the backward pass keeps two numbers a node and head and, of
    bfloat16, what the result's rounding left: where a node's weight is almost one, its gradient is what two such numbers leave."""
    kv_heads = num_heads if kv_heads is None else kv_heads
    _ops.check(q, k, v, graphs, num_heads, kv_heads, (before, after, sinks), scale)
    if scale is None:
        scale = (q.shape[1] * q.shape[2] // num_heads) ** -0.5
    args = q, k, v, graphs, num_heads, kv_heads, (before, after, sinks), float(scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _WindowAttention.apply(*args)
    return _ops.window_forward(*args, False)[0]


def window_attention_step(q: Tensor, keys: Tensor, values: Tensor, lengths: Tensor, num_heads: int, before: int, sinks: int = 0,
                          kv_heads: Optional[int] = None, scale: Optional[float] = None) -> Tensor:
    """The row of :func:`window_attention` (``after = 0``) of the last node of every chain, for chains that grow by a node at a time.

    ``q`` ``(chains, components, channels)`` is of the new nodes; ``keys`` and ``values`` ``(chains, capacity, components, kv channels)`` hold the chains so
    far, the new nodes among them, in their first ``lengths`` (chains,), int64, places; what lies behind is not read.  Lengths are read on the GPU, so the
    call can be captured in a CUDA graph and replayed while they grow; a length of zero gives zeros, one above the capacity counts as the capacity.
    Any strides but the channels'.  No gradients: inputs that need one are refused while gradients are recorded."""
    kv_heads = num_heads if kv_heads is None else kv_heads
    _ops.check_step(q, keys, values, lengths, num_heads, kv_heads, (before, sinks), scale)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, keys, values)):
        raise ValueError("a step has no gradient: call it under torch.no_grad() or detach the inputs")
    if scale is None:
        scale = (q.shape[1] * q.shape[2] // num_heads) ** -0.5
    return _ops.window_step(q, keys, values, lengths, num_heads, kv_heads, before, sinks, float(scale))
