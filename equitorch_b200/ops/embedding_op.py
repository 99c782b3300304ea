"""Rows of a table by type (operator layer over ``eqt_embedding_forward`` / ``eqt_embedding_grad``)."""
from __future__ import annotations

import math

import torch
from torch import Tensor

from .. import _lib


def check(index: Tensor, weight: Tensor) -> None:
    if weight.ndim < 2:
        raise ValueError(f"a table must be (types, ...) with at least one dimension of values, got {tuple(weight.shape)}")
    if weight.dtype not in _lib.DTYPE_CODE:
        raise TypeError(f"float32, float64 or bfloat16 table expected, got {weight.dtype}")
    if index.dtype != torch.int64:
        raise TypeError(f"int64 types expected, got {index.dtype}")


def embedding_forward(index: Tensor, weight: Tensor, scale: float) -> Tensor:
    """``out[..., :] = scale * weight[index[...], :]``; a row of zeros where ``index`` names no row of the table."""
    check(index, weight)
    dev = _lib.require_cuda(index, weight)
    index, weight = index.contiguous(), weight.contiguous()
    out = torch.empty(*index.shape, *weight.shape[1:], dtype=weight.dtype, device=dev)
    with _lib.on_device(dev):
        _lib.check(_lib.lib().eqt_embedding_forward(_lib.DTYPE_CODE[weight.dtype], weight.data_ptr(), index.data_ptr(), out.data_ptr(),
                                                    index.numel(), weight.shape[0], math.prod(weight.shape[1:]), scale,
                                                    _lib.stream_ptr(dev)), "eqt_embedding_forward")
    return out


def embedding_grad(index: Tensor, grad: Tensor, types: int, scale: float) -> Tensor:
    """``gw[t, :] = scale * sum of grad[n, :] over n with index[n] = t``: no atomics, sums in float32 (float64 for float64)."""
    row = grad.shape[index.ndim:]
    if grad.shape[:index.ndim] != index.shape:
        raise ValueError(f"gradient of shape {tuple(grad.shape)} for types of shape {tuple(index.shape)}")
    dev = _lib.require_cuda(index, grad)
    index, grad = index.contiguous(), grad.contiguous()
    n, width, code = index.numel(), math.prod(row), _lib.DTYPE_CODE[grad.dtype]
    gw = torch.empty(types, *row, dtype=grad.dtype, device=dev)
    with _lib.on_device(dev):                                # the size goes by the SMs of the current device
        size = _lib.lib().eqt_embedding_grad_scratch(code, n, types, width)
        scratch = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        _lib.check(_lib.lib().eqt_embedding_grad(code, grad.data_ptr(), index.data_ptr(), gw.data_ptr(), n, types, width, scale,
                                                 _lib.ptr(scratch), size, _lib.stream_ptr(dev)), "eqt_embedding_grad")
    return gw
