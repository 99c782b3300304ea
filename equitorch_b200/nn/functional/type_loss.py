"""Cross entropy over node types, without keeping the logits."""
from __future__ import annotations

from torch import Tensor
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from ...ops import type_loss_op as _ops


class _TypeCrossEntropy(Function):
    @staticmethod
    def forward(ctx, x, weight, target, reduction):
        loss, lse, count = _ops.loss_forward(x, weight, target, reduction)
        ctx.save_for_backward(x, weight, target, lse, count)
        ctx.reduction = reduction
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, target, lse, count = ctx.saved_tensors
        dx, dweight = _ops.loss_backward(grad, x, weight, target, ctx.reduction, lse, count, *ctx.needs_input_grad[:2])
        return dx, dweight, None, None


def type_cross_entropy(x: Tensor, weight: Tensor, target: Tensor, reduction: str = "mean") -> Tensor:
    r"""Cross entropy of the types that features ``x`` (..., channels) predict by a table ``weight`` (types, channels), as that of
    :func:`type_embedding`:

    .. math:: L_i = \log \sum_t \exp \langle x_i, w_t \rangle - \langle x_i, w_{target_i} \rangle

    ``target`` (...), int64.  Rows with a negative target do not count (nodes that are not masked, padding): their loss is zero, they have
    no gradient, and what their features hold reaches nothing.  A target that the table does not have gives NaN.  ``reduction``: ``mean`` over the rows
    that count (zero if none does), ``sum`` or ``none``; the loss is float32.

    float32 or bfloat16 features and table of one type, at most 16384 channels.  The logits are formed in tiles and never kept, once forward and once backward, where
    their gradients are in scratch for some types at a time (256 MB, or 128 types of over a million rows), beside a float32 sum of the size of ``x``
    and operands that are laid out anew (``x``; of float32 both, in three parts).  Sums in float32, no atomics; of bfloat16 the logits' gradients are rounded
    to bfloat16 for their products.  Differentiable once, in ``x`` and ``weight``."""
    _ops.check(x, weight, target, reduction)
    return _TypeCrossEntropy.apply(x, weight, target, reduction)
