"""Root-mean-square norm with the residual's addition (operator layer over ``eqt_add_rms_norm_forward`` / ``_e4m3`` / ``_backward``)."""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor

from .. import _lib


def check(x: Tensor, residual: Optional[Tensor], weight: Optional[Tensor], eps: float) -> None:
    if x.ndim not in (2, 3):
        raise ValueError(f"features must be (N, channels) or (N, components, channels), got {tuple(x.shape)}")
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"float32 or bfloat16 features expected, got {x.dtype}")
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"residual of shape {tuple(residual.shape)} for features of shape {tuple(x.shape)}")
    if weight is not None and tuple(weight.shape) != (x.shape[-1],):
        raise ValueError(f"weight of shape ({x.shape[-1]},) expected, got {tuple(weight.shape)}")
    for what, t in (("residual", residual), ("weight", weight)):
        if t is not None and t.dtype != x.dtype:
            raise TypeError(f"{what} of type {t.dtype} for features of type {x.dtype}")
    if not 1e-45 <= eps <= 3.4e38:                        # what float32 has
        raise ValueError(f"eps must be a positive float32, got {eps}")
    _lib.require_cuda(x, residual, weight)


def _sizes(x: Tensor) -> Tuple[int, int, int]:
    return x.shape[0], (x.shape[1] if x.ndim == 3 else 1), x.shape[-1]


def _whole(t: Optional[Tensor]) -> Optional[Tensor]:
    return None if t is None else t.contiguous()


def norm_forward(x: Tensor, residual: Optional[Tensor], weight: Optional[Tensor], eps: float, want_stats: bool
                 ) -> Tuple[Tensor, Tensor, Optional[Tensor]]:
    """The normalised sum, the sum (``x`` itself without a residual) and, where wanted, the nodes' inverse roots."""
    dev = x.device
    given, x, residual, weight = x, _whole(x), _whole(residual), _whole(weight)
    n, comps, channels = _sizes(x)
    out = torch.empty_like(x)
    total = given.view_as(given) if residual is None else torch.empty_like(x)
    rstd = torch.empty(n, dtype=torch.float32, device=dev) if want_stats else None
    with _lib.on_device(dev):
        _lib.check(_lib.lib().eqt_add_rms_norm_forward(_lib.DTYPE_CODE[x.dtype], x.data_ptr(), _lib.ptr(residual), _lib.ptr(weight), out.data_ptr(),
                                                       None if residual is None else total.data_ptr(), _lib.ptr(rstd), n, comps, channels, eps,
                                                       _lib.stream_ptr(dev)), "eqt_add_rms_norm_forward")
    return out, total, rstd


def norm_e4m3(x: Tensor, residual: Optional[Tensor], weight: Optional[Tensor], eps: float, group: int) -> Tuple[Tensor, Tensor, Tensor]:
    """8-bit values, their scales ``(N, groups)`` and the sum."""
    dev = x.device
    given, x, residual, weight = x, _whole(x), _whole(residual), _whole(weight)
    n, comps, channels = _sizes(x)
    values = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=dev)
    scales = torch.empty(n, comps * channels // group, dtype=torch.float32, device=dev)
    total = given if residual is None else torch.empty_like(x)
    with _lib.on_device(dev):
        _lib.check(_lib.lib().eqt_add_rms_norm_e4m3(_lib.DTYPE_CODE[x.dtype], x.data_ptr(), _lib.ptr(residual), _lib.ptr(weight), values.data_ptr(),
                                                    scales.data_ptr(), None if residual is None else total.data_ptr(), n, comps, channels, group, eps,
                                                    _lib.stream_ptr(dev)), "eqt_add_rms_norm_e4m3")
    return values, scales, total


def norm_backward(grad: Tensor, grad_total: Optional[Tensor], total: Tensor, residual: Optional[Tensor], weight: Optional[Tensor], rstd: Tensor,
                  want_weight: bool) -> Tuple[Tensor, Optional[Tensor]]:
    """The gradient of the features, which is the residual's too, and that of the weight; the sum is ``total``, or that of both."""
    dev = total.device
    grad, grad_total, total, residual, weight = _whole(grad), _whole(grad_total), _whole(total), _whole(residual), _whole(weight)
    n, comps, channels = _sizes(total)
    dx = torch.empty_like(total)
    dweight = torch.empty_like(weight) if want_weight else None
    code, lib = _lib.DTYPE_CODE[total.dtype], _lib.lib()
    with _lib.on_device(dev):
        size = lib.eqt_add_rms_norm_scratch(code, n, comps, channels) if want_weight else 0
        scratch = torch.empty(size, dtype=torch.float32, device=dev) if size else None
        _lib.check(lib.eqt_add_rms_norm_backward(code, grad.data_ptr(), _lib.ptr(grad_total), total.data_ptr(), _lib.ptr(residual), _lib.ptr(weight),
                                                 rstd.data_ptr(), dx.data_ptr(), _lib.ptr(dweight), _lib.ptr(scratch), size, n, comps, channels, _lib.stream_ptr(dev)),
                   "eqt_add_rms_norm_backward")
    return dx, dweight
