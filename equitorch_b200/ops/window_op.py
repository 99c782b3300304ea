"""Attention within windows of chains (operator layer over ``eqt_window_attention_*`` and ``eqt_window_step``)."""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch
from torch import Tensor

from .. import _lib
from ..graph import PackedGraphs
from .attention_op import MAX_HEAD
from .fused_tp_op import status_flag


def _check_heads(q: Tensor, k: Tensor, v: Tensor, heads: int, kv_heads: int, window: Tuple[int, ...], scale: Optional[float]) -> None:
    if k.shape != v.shape:
        raise ValueError(f"k and v must have the same shape, got {tuple(k.shape)} and {tuple(v.shape)}")
    if q.dtype not in (torch.float32, torch.bfloat16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"float32 or bfloat16 features of one type expected, got {q.dtype}, {k.dtype} and {v.dtype}")
    if heads < 1 or kv_heads < 1 or heads % kv_heads:
        raise ValueError(f"{heads} heads cannot share {kv_heads} heads of keys")
    if q.shape[-1] == 0 or q.shape[-2] == 0 or q.shape[-1] % heads or k.shape[-1] != q.shape[-1] // heads * kv_heads or k.shape[-2] != q.shape[-2]:
        raise ValueError(f"{heads} heads of queries of shape {tuple(q.shape)} and {kv_heads} of keys of shape {tuple(k.shape)} do not go together")
    if q.shape[-2] * q.shape[-1] // heads > MAX_HEAD:
        raise ValueError(f"a head has at most {MAX_HEAD} values a node: {q.shape[-2]} components of {q.shape[-1] // heads} channels are more")
    if any(not isinstance(w, int) or not 0 <= w < 2 ** 31 for w in window):
        raise ValueError(f"windows and sinks are whole numbers in [0, 2^31), got {window}")
    if scale is not None and not abs(scale) <= 1e12:
        raise ValueError(f"the scale must be at most 1e12, got {scale}")


def check(q: Tensor, k: Tensor, v: Tensor, graphs: PackedGraphs, heads: int, kv_heads: int, window: Tuple[int, ...], scale: Optional[float]) -> None:
    if not isinstance(graphs, PackedGraphs):
        raise TypeError(f"PackedGraphs expected, got {type(graphs).__name__}")
    if q.ndim != 3 or k.ndim != 3:
        raise ValueError(f"features must be (N, components, channels), got {tuple(q.shape)} and {tuple(k.shape)}")
    _check_heads(q, k, v, heads, kv_heads, window, scale)
    if q.shape[0] != graphs.num_nodes or k.shape[0] != graphs.num_nodes:
        raise ValueError(f"the graphs have {graphs.num_nodes} nodes, the features {q.shape[0]} and {k.shape[0]}")
    _lib.require_cuda(q, k, v, graphs.tiles)


def check_step(q: Tensor, keys: Tensor, values: Tensor, lengths: Tensor, heads: int, kv_heads: int, window: Tuple[int, ...], scale: Optional[float]) -> None:
    if q.ndim != 3 or keys.ndim != 4:
        raise ValueError(f"queries (chains, components, channels) and a cache (chains, capacity, components, channels) expected, got {tuple(q.shape)} "
                         f"and {tuple(keys.shape)}")
    _check_heads(q, keys, values, heads, kv_heads, window, scale)
    if keys.shape[0] != q.shape[0] or tuple(lengths.shape) != (q.shape[0],):
        raise ValueError(f"{q.shape[0]} chains of queries, {keys.shape[0]} of keys and lengths of shape {tuple(lengths.shape)}")
    if lengths.dtype != torch.int64:
        raise TypeError(f"int64 lengths expected, got {lengths.dtype}")
    _lib.require_cuda(q, keys, values, lengths)


def _rows(x: Tensor) -> Tensor:
    """The kernels take any strides but the channels', which are next to each other."""
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _args(q, k, v, graphs, heads, kv_heads, window, scale, out, rest, stats) -> _lib.WindowAttentionArgs:
    n, comps, channels = q.shape
    return _lib.WindowAttentionArgs(
        dtype=_lib.DTYPE_CODE[q.dtype], comps=comps, heads=heads, kv_heads=kv_heads, head_channels=channels // heads, tile_rows=graphs.tile_rows,
        scale=scale, n=n, num_graphs=graphs.num_graphs, longest=graphs.longest, num_tiles=graphs.tiles.shape[0], before=window[0], after=window[1],
        sinks=window[2], q_node=q.stride(0), q_comp=q.stride(1), k_node=k.stride(0), k_comp=k.stride(1), v_node=v.stride(0), v_comp=v.stride(1),
        ptr=graphs.ptr.data_ptr(), tiles=graphs.tiles.data_ptr(), q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(),
        rest=_lib.ptr(rest), stats=_lib.ptr(stats), status=status_flag(q.device).data_ptr())


def _new(like: Tensor, graphs: PackedGraphs) -> Tensor:
    """A result of the shape of ``like``; rows of no graph are zero."""
    return (torch.empty if graphs.covers else torch.zeros)(like.shape, dtype=like.dtype, device=like.device)


def _scratch(args: _lib.WindowAttentionArgs, backward: bool, dev: torch.device) -> Optional[Tensor]:
    size = _lib.lib().eqt_window_attention_scratch(C.byref(args), int(backward))
    scratch = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    args.scratch, args.scratch_bytes = _lib.ptr(scratch), size
    return scratch


def window_forward(q: Tensor, k: Tensor, v: Tensor, graphs: PackedGraphs, heads: int, kv_heads: int, window: Tuple[int, int, int], scale: float,
                   want_stats: bool) -> Tuple[Tensor, Optional[Tensor], Optional[Tensor]]:
    """The result and, for the backward pass, what its rounding left (of bfloat16) and the rows' statistics."""
    dev = q.device
    q, k, v = _rows(q), _rows(k), _rows(v)
    out = _new(q, graphs)
    rest = _new(q, graphs) if want_stats and q.dtype == torch.bfloat16 else None
    stats = torch.empty(2, heads, q.shape[0], dtype=torch.float32, device=dev) if want_stats else None
    args = _args(q, k, v, graphs, heads, kv_heads, window, scale, out, rest, stats)
    with _lib.on_device(dev):
        scratch = _scratch(args, False, dev)  # noqa: F841 - kept alive for the call
        _lib.check(_lib.lib().eqt_window_attention_forward(C.byref(args), _lib.stream_ptr(dev)), "eqt_window_attention_forward")
    return out, rest, stats


def window_backward(grad: Tensor, q: Tensor, k: Tensor, v: Tensor, graphs: PackedGraphs, heads: int, kv_heads: int, window: Tuple[int, int, int],
                    scale: float, out: Tensor, rest: Optional[Tensor], stats: Tensor) -> Tuple[Tensor, Tensor, Tensor]:
    dev = q.device
    q, k, v, grad = _rows(q), _rows(k), _rows(v), grad.contiguous()
    dq, dk, dv = _new(q, graphs), _new(k, graphs), _new(k, graphs)
    args = _args(q, k, v, graphs, heads, kv_heads, window, scale, out, rest, stats)
    args.grad, args.dq, args.dk, args.dv = grad.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
    with _lib.on_device(dev):
        scratch = _scratch(args, True, dev)  # noqa: F841 - kept alive for the call
        _lib.check(_lib.lib().eqt_window_attention_backward(C.byref(args), _lib.stream_ptr(dev)), "eqt_window_attention_backward")
    return dq, dk, dv


def window_step(q: Tensor, keys: Tensor, values: Tensor, lengths: Tensor, heads: int, kv_heads: int, before: int, sinks: int, scale: float) -> Tensor:
    dev = q.device
    q, keys, values, lengths = _rows(q), _rows(keys), _rows(values), lengths.contiguous()
    out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    args = _lib.WindowStepArgs(
        dtype=_lib.DTYPE_CODE[q.dtype], comps=q.shape[1], heads=heads, kv_heads=kv_heads, head_channels=q.shape[2] // heads, scale=scale,
        chains=q.shape[0], capacity=keys.shape[1], before=before, sinks=sinks, q_chain=q.stride(0), q_comp=q.stride(1), k_chain=keys.stride(0),
        k_node=keys.stride(1), k_comp=keys.stride(2), v_chain=values.stride(0), v_node=values.stride(1), v_comp=values.stride(2), q=q.data_ptr(),
        k=keys.data_ptr(), v=values.data_ptr(), out=out.data_ptr(), lengths=lengths.data_ptr())
    with _lib.on_device(dev):
        size = _lib.lib().eqt_window_step_scratch(C.byref(args))
        scratch = torch.empty(size, dtype=torch.float32, device=dev) if size else None
        args.scratch, args.scratch_floats = _lib.ptr(scratch), size
        _lib.check(_lib.lib().eqt_window_step(C.byref(args), _lib.stream_ptr(dev)), "eqt_window_step")
    return out
