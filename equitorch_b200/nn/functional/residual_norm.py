"""Root-mean-square norm of a node's values with the residual's addition before it."""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from ...ops import residual_norm_op as _ops


class _AddRMSNorm(Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        out, total, rstd = _ops.norm_forward(x, residual, weight, eps, any(ctx.needs_input_grad))
        apart = residual is not None and x.dtype == torch.bfloat16
        ctx.save_for_backward(x if residual is None or apart else total, residual if apart else None, weight, rstd)
        ctx.set_materialize_grads(False)
        return out, total

    @staticmethod
    @once_differentiable
    def backward(ctx, grad, grad_total):
        total, residual, weight, rstd = ctx.saved_tensors
        need_x, need_residual, need_weight, _ = ctx.needs_input_grad
        if grad is None:                                 # only the sum was used
            dx, dweight = grad_total, torch.zeros_like(weight) if need_weight else None
        else:
            dx, dweight = _ops.norm_backward(grad, grad_total, total, residual, weight, rstd, need_weight)
        return dx if need_x else None, dx if need_residual else None, dweight, None


def add_rms_norm(x: Tensor, residual: Optional[Tensor] = None, weight: Optional[Tensor] = None, eps: float = 1e-6) -> Tuple[Tensor, Tensor]:
    r"""The norm in front of a transformer's block, with the addition of the block before: both the normalised sum and the sum, which is the
    residual of the next call:

    .. math:: h = x + residual, \quad out = h / \sqrt{mean(h^2) + eps} * weight

    ``x`` and ``residual`` (or ``None``: the sum is ``x`` itself) are ``(N, channels)`` or ``(N, components, channels)``; the mean is over all
    of a node's components and channels and ``weight`` (channels,) has no components, so equivariant features stay so.  float32 or bfloat16, all of one
    type; sums in float32.  ``out`` is computed from the sum before its rounding.  Kept for the backward pass are one number a node and the sum, or, of
    bfloat16, ``x`` and ``residual``, since the sum's rounding would go into the gradients beside their own.

    Differentiable once, in ``x``, ``residual`` and ``weight``; the weight's gradient uses no atomics and is the same bits at every call."""
    _ops.check(x, residual, weight, eps)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight)):
        return _AddRMSNorm.apply(x, residual, weight, float(eps))
    return _ops.norm_forward(x, residual, weight, float(eps), False)[:2]


def add_rms_norm_e4m3(x: Tensor, residual: Optional[Tensor] = None, weight: Optional[Tensor] = None, eps: float = 1e-6, group: Optional[int] = None
                      ) -> Tuple[Tensor, Tensor, Tensor]:
    """:func:`add_rms_norm` for a product in 8 bits at inference: ``values`` (float8_e4m3fn, of the shape of ``x``), ``scales`` (float32,
    ``(N, groups)``) and the sum.  Every ``group`` values of a node (a divisor of components times channels; all of them where not given) share a
    scale, which brings the greatest of them to 448, the greatest number of the type; ``out = values * scale``.  The values are the nearest
    to the exact quotients, ties to even.  A group of zeros has the scale zero.  Values that are not finite, or whose squares' sum is not in
    float32, make all of the node's scales NaN, weights that are not finite all nodes'.  No gradients: inputs that need one are refused while gradients are recorded."""
    _ops.check(x, residual, weight, eps)
    values = x.shape[-1] * (x.shape[1] if x.ndim == 3 else 1)
    if group is not None and (group < 1 or values % group):
        raise ValueError(f"groups of {group} do not divide {values} values a node")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, weight)):
        raise ValueError("the result in 8 bits has no gradient: call it under torch.no_grad() or detach the inputs")
    return _ops.norm_e4m3(x, residual, weight, float(eps), max(1, values) if group is None else int(group))
