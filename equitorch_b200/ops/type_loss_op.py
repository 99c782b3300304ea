"""Cross entropy over types (operator layer over ``eqt_type_loss_forward`` / ``eqt_type_loss_backward``)."""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch
from torch import Tensor

from .. import _lib
from .fused_tp_op import status_flag

REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def check(x: Tensor, weight: Tensor, target: Tensor, reduction: str) -> None:
    if reduction not in REDUCTIONS:
        raise ValueError(f"reduction should be in {list(REDUCTIONS)}, got {reduction}")
    if weight.ndim != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"a table of (types, channels) expected, got {tuple(weight.shape)}")
    if x.ndim < 1 or x.shape[-1] != weight.shape[1] or target.shape != x.shape[:-1]:
        raise ValueError(f"features (..., {weight.shape[1]}) and a type for each row expected, got {tuple(x.shape)} and {tuple(target.shape)}")
    if x.dtype not in (torch.float32, torch.bfloat16) or weight.dtype != x.dtype:
        raise TypeError(f"features and table of one type of float32 and bfloat16 expected, got {x.dtype} and {weight.dtype}")
    if target.dtype != torch.int64:
        raise TypeError(f"int64 types expected, got {target.dtype}")
    _lib.require_cuda(x, weight, target)


def _aligned(t: Tensor) -> Tensor:
    """Contiguous and, as the copies of tiles need it, on a 16-byte boundary."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _args(x, weight, target, reduction, lse, count) -> _lib.TypeLossArgs:
    return _lib.TypeLossArgs(dtype=_lib.DTYPE_CODE[x.dtype], reduction=REDUCTIONS[reduction], n=target.numel(), c=weight.shape[1], t=weight.shape[0],
                             x=x.data_ptr(), w=weight.data_ptr(), target=target.data_ptr(), lse=lse.data_ptr(), count=count.data_ptr(),
                             status=status_flag(x.device).data_ptr())


def _scratch(args: _lib.TypeLossArgs, backward: bool, dev: torch.device) -> Optional[Tensor]:
    size = _lib.lib().eqt_type_loss_scratch(C.byref(args), int(backward))
    scratch = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    args.scratch, args.scratch_bytes = _lib.ptr(scratch), size
    return scratch


def loss_forward(x: Tensor, weight: Tensor, target: Tensor, reduction: str) -> Tuple[Tensor, Tensor, Tensor]:
    """The loss (of every row, or one number), the rows' log sums (in units of log2) and how many rows count; all float32."""
    dev = x.device
    x, weight, target = _aligned(x), _aligned(weight), target.contiguous()
    losses = torch.empty(target.shape, dtype=torch.float32, device=dev)
    lse, count = torch.empty(target.numel(), dtype=torch.float32, device=dev), torch.empty(1, dtype=torch.float32, device=dev)
    result = None if reduction == "none" else torch.empty((), dtype=torch.float32, device=dev)
    args = _args(x, weight, target, reduction, lse, count)
    args.losses, args.result = losses.data_ptr(), _lib.ptr(result)
    with _lib.on_device(dev):
        scratch = _scratch(args, False, dev)  # noqa: F841 - kept alive for the call
        _lib.check(_lib.lib().eqt_type_loss_forward(C.byref(args), _lib.stream_ptr(dev)), "eqt_type_loss_forward")
    return losses if result is None else result, lse, count


def loss_backward(grad: Tensor, x: Tensor, weight: Tensor, target: Tensor, reduction: str, lse: Tensor, count: Tensor, want_x: bool, want_weight: bool
                  ) -> Tuple[Optional[Tensor], Optional[Tensor]]:
    dev = x.device
    x, weight, target, grad = _aligned(x), _aligned(weight), target.contiguous(), grad.contiguous()
    dx = torch.empty_like(x) if want_x else None
    dw = torch.empty_like(weight) if want_weight else None
    args = _args(x, weight, target, reduction, lse, count)
    args.grad, args.dx, args.dw = grad.data_ptr(), _lib.ptr(dx), _lib.ptr(dw)
    with _lib.on_device(dev):
        scratch = _scratch(args, True, dev)  # noqa: F841 - kept alive for the call
        _lib.check(_lib.lib().eqt_type_loss_backward(C.byref(args), _lib.stream_ptr(dev)), "eqt_type_loss_backward")
    return dx, dw
