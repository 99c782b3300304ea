"""Features by node or edge type: the first layer of a network over typed nodes."""
from __future__ import annotations

import torch
from torch import Tensor
from torch.autograd import Function

from ...ops import embedding_op as _ops


class _Embedding(Function):
    @staticmethod
    def forward(ctx, weight: Tensor, index: Tensor, scale: float) -> Tensor:
        ctx.save_for_backward(index)
        ctx.types, ctx.scale = weight.shape[0], scale
        return _ops.embedding_forward(index, weight, scale)

    @staticmethod
    def backward(ctx, grad: Tensor):
        (index,) = ctx.saved_tensors
        adjoint = _EmbeddingGrad.apply if torch.is_grad_enabled() else _ops_grad
        return adjoint(grad, index, ctx.types, ctx.scale), None, None


class _EmbeddingGrad(Function):
    """The adjoint of the lookup (and the lookup is its adjoint)."""

    @staticmethod
    def forward(ctx, grad: Tensor, index: Tensor, types: int, scale: float) -> Tensor:
        ctx.save_for_backward(index)
        ctx.scale = scale
        return _ops_grad(grad, index, types, scale)

    @staticmethod
    def backward(ctx, g: Tensor):
        return _Embedding.apply(g, ctx.saved_tensors[0], ctx.scale), None, None, None


def _ops_grad(grad: Tensor, index: Tensor, types: int, scale: float) -> Tensor:
    return _ops.embedding_grad(index, grad, types, scale)


def type_embedding(index: Tensor, weight: Tensor, scale: float = 1.0) -> Tensor:
    """``out[..., :] = scale * weight[index[...], :]`` for ``index`` of any shape (int64) and a table ``weight`` of shape
    ``(types, ...)``; the result is ``(*index.shape, *weight.shape[1:])`` in the table's type.

    An index outside ``[0, types)`` (a padded node, say) gives a row of zeros and no gradient.  The gradient of the table has
    its sums in float32 (float64 for float64), uses no atomics and is the same bits at every call; both directions can be
    differentiated again and captured in a CUDA graph."""
    return _Embedding.apply(weight, index, float(scale))
