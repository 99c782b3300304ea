"""Rotary positions (operator layer over ``eqt_rotary``)."""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch
from torch import Tensor

from .. import _lib


def check(q: Tensor, k: Optional[Tensor], positions: Tensor, frequencies: Tensor, heads: int, kv_heads: int) -> None:
    for x, h in ((q, heads), (k, kv_heads)):
        if x is None:
            continue
        if x.ndim != 3:
            raise ValueError(f"features must be (N, components, channels), got {tuple(x.shape)}")
        if h < 1 or x.shape[2] % h or x.shape[2] == 0:
            raise ValueError(f"{h} heads cannot share features of shape {tuple(x.shape)}")
    if q.dtype not in (torch.float32, torch.bfloat16) or (k is not None and k.dtype != q.dtype):
        raise TypeError(f"float32 or bfloat16 features of one type expected, got {q.dtype}" + ("" if k is None else f" and {k.dtype}"))
    size = q.shape[2] // heads
    if k is not None and (k.shape[:2] != q.shape[:2] or k.shape[2] // kv_heads != size):
        raise ValueError(f"k of shape {tuple(k.shape)} with {kv_heads} heads does not go with q of shape {tuple(q.shape)} with {heads}")
    if positions.dtype != torch.int64 or frequencies.dtype != torch.float64:
        raise TypeError(f"int64 positions and float64 frequencies expected, got {positions.dtype} and {frequencies.dtype}")
    if tuple(positions.shape) != (q.shape[0],):
        raise ValueError(f"positions ({q.shape[0]},) expected, got {tuple(positions.shape)}")
    if frequencies.ndim != 1 or 2 * frequencies.shape[0] > size:
        raise ValueError(f"frequencies of at most {size // 2} pairs of a head's {size} channels expected, got {tuple(frequencies.shape)}")
    _lib.require_cuda(q, k, positions, frequencies)


def _rows(x: Optional[Tensor]) -> Optional[Tensor]:
    """The kernels take any strides of nodes and components; channels are next to each other."""
    return x if x is None or x.stride(2) == 1 or x.shape[2] == 1 else x.contiguous()


def rotary(q: Tensor, k: Optional[Tensor], positions: Tensor, frequencies: Tensor, heads: int, kv_heads: int, interleaved: bool, magnitude: float,
           backward: bool) -> Tuple[Tensor, Optional[Tensor]]:
    dev = q.device
    q, k, positions, frequencies = _rows(q), _rows(k), positions.contiguous(), frequencies.contiguous()
    out = [None if x is None else torch.empty(x.shape, dtype=x.dtype, device=dev) for x in (q, k)]
    args = _lib.RotaryArgs(dtype=_lib.DTYPE_CODE[q.dtype], comps=q.shape[1], heads=heads, kv_heads=kv_heads, size=q.shape[2] // heads,
                           half=frequencies.shape[0], interleaved=interleaved, backward=backward, magnitude=magnitude, n=q.shape[0],
                           q_node=q.stride(0), q_comp=q.stride(1), q=q.data_ptr(), q_out=out[0].data_ptr(), positions=positions.data_ptr(),
                           frequencies=frequencies.data_ptr())
    if k is not None:
        args.k_node, args.k_comp, args.k, args.k_out = k.stride(0), k.stride(1), k.data_ptr(), out[1].data_ptr()
    with _lib.on_device(dev):
        _lib.check(_lib.lib().eqt_rotary(C.byref(args), _lib.stream_ptr(dev)), "eqt_rotary")
    return out[0], out[1]
