"""Attention within packed graphs (operator layer over ``eqt_attention_forward`` / ``eqt_attention_backward``)."""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch
from torch import Tensor

from .. import _lib
from ..graph import PackedGraphs

#: values of a head at one node that the kernels hold
MAX_HEAD = 128


def check(q: Tensor, k: Tensor, v: Tensor, graphs: PackedGraphs, heads: int, scale: Optional[float], cap: Optional[float],
          pos: Optional[Tensor], slope: Optional[Tensor]) -> None:
    if not isinstance(graphs, PackedGraphs):
        raise TypeError(f"PackedGraphs expected, got {type(graphs).__name__}")
    if q.ndim != 3:
        raise ValueError(f"features must be (N, components, channels), got {tuple(q.shape)}")
    if q.shape != k.shape or q.shape != v.shape:
        raise ValueError(f"q, k and v must have the same shape, got {tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
    if q.dtype not in (torch.float32, torch.bfloat16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"float32 or bfloat16 features of one type expected, got {q.dtype}, {k.dtype} and {v.dtype}")
    if q.shape[0] != graphs.num_nodes:
        raise ValueError(f"the graphs have {graphs.num_nodes} nodes, the features {q.shape[0]}")
    if heads < 1 or q.shape[2] % heads or q.shape[2] == 0 or q.shape[1] == 0:
        raise ValueError(f"{heads} heads cannot share features of shape {tuple(q.shape)}")
    if q.shape[1] * q.shape[2] // heads > MAX_HEAD:
        raise ValueError(f"a head has at most {MAX_HEAD} values a node: {q.shape[1]} components of {q.shape[2] // heads} channels are more")
    if cap is not None and not 1e-12 <= cap <= 1e12:
        raise ValueError(f"the cap must be from 1e-12 to 1e12, got {cap}")
    if scale is not None and not abs(scale) <= 1e12:
        raise ValueError(f"the scale must be at most 1e12, got {scale}")
    if (pos is None) != (slope is None):
        raise ValueError("positions and slopes come together")
    if pos is not None:
        if tuple(pos.shape) != (q.shape[0], 3) or tuple(slope.shape) != (heads,):
            raise ValueError(f"positions ({q.shape[0]}, 3) and slopes ({heads},) expected, got {tuple(pos.shape)} and {tuple(slope.shape)}")
        if pos.dtype != torch.float32 or slope.dtype != torch.float32:
            raise TypeError(f"float32 positions and slopes expected, got {pos.dtype} and {slope.dtype}")
    _lib.require_cuda(q, k, v, pos, slope, graphs.tiles)


def _rows(x: Tensor) -> Tensor:
    """The kernels take any strides of nodes and components; channels are next to each other."""
    return x if x.stride(2) == 1 or x.shape[2] == 1 else x.contiguous()


def _args(q, k, v, graphs, heads, scale, cap, pos, slope, out, stats) -> _lib.AttentionArgs:
    n, comps, channels = q.shape
    return _lib.AttentionArgs(
        dtype=_lib.DTYPE_CODE[q.dtype], heads=heads, comps=comps, head_channels=channels // heads, tile_rows=graphs.tile_rows,
        scale=scale, cap=cap or 0.0, n=n, longest=graphs.longest, num_tiles=graphs.tiles.shape[0], tiles=graphs.tiles.data_ptr(),
        q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), q_node=q.stride(0), q_comp=q.stride(1), k_node=k.stride(0),
        k_comp=k.stride(1), v_node=v.stride(0), v_comp=v.stride(1), pos=_lib.ptr(pos), slope=_lib.ptr(slope),
        out=out.data_ptr(), stats=_lib.ptr(stats))


def _new(like: Tensor, graphs: PackedGraphs) -> Tensor:
    """A result of the shape of ``like``; rows of no graph are zero."""
    return (torch.empty if graphs.covers else torch.zeros)(like.shape, dtype=like.dtype, device=like.device)


def attention_forward(q: Tensor, k: Tensor, v: Tensor, graphs: PackedGraphs, heads: int, scale: float, cap: Optional[float],
                      pos: Optional[Tensor], slope: Optional[Tensor], want_stats: bool) -> Tuple[Tensor, Optional[Tensor]]:
    dev = q.device
    q, k, v = _rows(q), _rows(k), _rows(v)
    pos, slope = (None, None) if pos is None else (pos.contiguous(), slope.contiguous())
    out = _new(q, graphs)
    stats = torch.empty(2, heads, q.shape[0], dtype=torch.float32, device=dev) if want_stats else None
    args = _args(q, k, v, graphs, heads, scale, cap, pos, slope, out, stats)
    with _lib.on_device(dev):
        _lib.check(_lib.lib().eqt_attention_forward(C.byref(args), _lib.stream_ptr(dev)), "eqt_attention_forward")
    return out, stats


def attention_backward(grad: Tensor, q: Tensor, k: Tensor, v: Tensor, graphs: PackedGraphs, heads: int, scale: float,
                       cap: Optional[float], pos: Optional[Tensor], slope: Optional[Tensor], out: Tensor, stats: Tensor,
                       want_geometry: bool):
    """Gradients of q, k, v and, where wanted, of the slopes and positions (else ``None``)."""
    dev = q.device
    q, k, v, grad = _rows(q), _rows(k), _rows(v), grad.contiguous()
    pos, slope = (None, None) if pos is None else (pos.contiguous(), slope.contiguous())
    dq, dk, dv = _new(q, graphs), _new(q, graphs), _new(q, graphs)
    args = _args(q, k, v, graphs, heads, scale, cap, pos, slope, out, stats)
    args.grad_out, args.dq, args.dk, args.dv = grad.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
    dslope = dpos = None
    rows = heads * q.shape[0]                             # of scratch: eight numbers of geometry and one of the softmax's gradient each
    scratch = (torch.empty if graphs.covers else torch.zeros)(rows * (9 if want_geometry else 1), dtype=torch.float32, device=dev)
    args.delta = scratch.data_ptr() + 4 * (scratch.numel() - rows)
    if want_geometry:
        dslope, dpos = torch.empty_like(slope), torch.empty_like(pos)
        args.geo, args.dpos, args.dslope = scratch.data_ptr(), dpos.data_ptr(), dslope.data_ptr()
    with _lib.on_device(dev):
        _lib.check(_lib.lib().eqt_attention_backward(C.byref(args), _lib.stream_ptr(dev)), "eqt_attention_backward")
    return dq, dk, dv, dslope, dpos
