"""Gated linear layer (operator layer over ``eqt_gated_forward`` / ``eqt_gated_backward``)."""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor

from .. import _lib
from .fused_tp_op import status_flag

ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2, "sigmoid": 3}


def check(x: Tensor, weight: Tensor, activation: str) -> None:
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation should be in {list(ACTIVATIONS)}, got {activation}")
    if weight.ndim != 3 or weight.shape[0] != 2:
        raise ValueError(f"weight must be (2, channels, hidden), got {tuple(weight.shape)}")
    if x.ndim < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"features (..., {weight.shape[1]}) expected, got {tuple(x.shape)}")
    if x.dtype not in _lib.DTYPE_CODE or weight.dtype != x.dtype:
        raise TypeError(f"features and weight of one type of float32, float64 and bfloat16 expected, got {x.dtype} and {weight.dtype}")
    _lib.require_cuda(x, weight)


def _aligned(t: Tensor) -> Tensor:
    """Contiguous and, as the copies of tiles need it, on a 16-byte boundary."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def gated_forward(x: Tensor, weight: Tensor, activation: str) -> Tensor:
    """``act(x @ weight[0]) * (x @ weight[1])`` over the last dimension of ``x``."""
    dev = x.device
    x, weight = _aligned(x), _aligned(weight)
    c, f = weight.shape[1:]
    h = torch.empty(*x.shape[:-1], f, dtype=x.dtype, device=dev)
    n = h.numel() // f if f else 0
    code, lib = _lib.DTYPE_CODE[x.dtype], _lib.lib()
    with _lib.on_device(dev):
        size = lib.eqt_gated_scratch(code, n, c, f, 0)
        scratch = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        _lib.check(lib.eqt_gated_forward(code, x.data_ptr(), weight.data_ptr(), h.data_ptr(), _lib.ptr(scratch), size, n, c, f,
                                         ACTIVATIONS[activation], status_flag(dev).data_ptr(), _lib.stream_ptr(dev)), "eqt_gated_forward")
    return h


def gated_backward(grad: Tensor, x: Tensor, weight: Tensor, activation: str, want_x: bool, want_weight: bool
                   ) -> Tuple[Optional[Tensor], Optional[Tensor]]:
    dev = x.device
    x, weight, grad = _aligned(x), _aligned(weight), _aligned(grad)
    c, f = weight.shape[1:]
    n = x.numel() // c if c else 0
    dx = torch.empty_like(x) if want_x else None
    dw = torch.empty_like(weight) if want_weight else None
    code, lib = _lib.DTYPE_CODE[x.dtype], _lib.lib()
    with _lib.on_device(dev):
        size = lib.eqt_gated_scratch(code, n, c, f, 1)
        scratch = torch.empty(size, dtype=torch.uint8, device=dev)
        _lib.check(lib.eqt_gated_backward(code, x.data_ptr(), weight.data_ptr(), grad.data_ptr(), _lib.ptr(dx), _lib.ptr(dw),
                                          scratch.data_ptr(), size, n, c, f, ACTIVATIONS[activation], status_flag(dev).data_ptr(),
                                          _lib.stream_ptr(dev)), "eqt_gated_backward")
    return dx, dw
