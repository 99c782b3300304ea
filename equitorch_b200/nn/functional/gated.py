"""Gated linear layer: two projections, the activation of one and their product."""
from __future__ import annotations

from torch import Tensor
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from ...ops import gated_op as _ops


class _GatedLinear(Function):
    @staticmethod
    def forward(ctx, x: Tensor, weight: Tensor, activation: str) -> Tensor:
        ctx.save_for_backward(x, weight)
        ctx.activation = activation
        return _ops.gated_forward(x, weight, activation)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad: Tensor):
        x, weight = ctx.saved_tensors
        dx, dw = _ops.gated_backward(grad, x, weight, ctx.activation, *ctx.needs_input_grad[:2])
        return dx, dw, None


def gated_linear(input: Tensor, weight: Tensor, activation: str = "silu") -> Tensor:
    """``act(x W[0]) * (x W[1])`` for features ``x`` of shape ``(..., channels)`` and a weight of shape ``(2, channels, hidden)``:
    the first half of a gated feed-forward block, in one kernel.  ``activation`` is ``silu``, ``gelu`` (the one with the error
    function), ``relu`` or ``sigmoid``; of equivariant features it may act on invariant components only.

    float32, float64 or bfloat16, sums in float32 (float64 for float64).  Differentiable once (no training on forces through it); the backward pass forms both
    projections again, keeps only ``x`` and the weight, and takes scratch of twice the result's size.  float32 and bfloat16 run on
    the tensor cores; where channels or hidden are no multiples of 16 bytes (4 or 8 values) the operands are first copied to wider
    rows."""
    _ops.check(input, weight, activation)
    return _GatedLinear.apply(input, weight, activation)
