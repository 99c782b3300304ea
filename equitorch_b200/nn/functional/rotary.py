"""Rotary positions: where a node is along its chain, as turns of channel pairs."""
from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch
from torch import Tensor
from torch.autograd import Function

from ...ops import rotary_op as _ops


class _Rotary(Function):
    """Its adjoint is itself the other way round, so it can be differentiated as often as one likes."""

    @staticmethod
    def forward(ctx, q, k, positions, frequencies, heads, kv_heads, interleaved, magnitude, backward):
        ctx.save_for_backward(positions, frequencies)
        ctx.args = heads, kv_heads, interleaved, magnitude
        ctx.turned_back = backward
        return _ops.rotary(q, k, positions, frequencies, heads, kv_heads, interleaved, magnitude, backward)

    @staticmethod
    def backward(ctx, dq, dk):
        positions, frequencies = ctx.saved_tensors
        dq, dk = _Rotary.apply(dq, dk if ctx.needs_input_grad[1] else None, positions, frequencies, *ctx.args, not ctx.turned_back)
        return (dq if ctx.needs_input_grad[0] else None, dk if ctx.needs_input_grad[1] else None, *[None] * 7)


def rotary_frequencies(rotated: int, base: float = 10_000.0, factor: float = 1.0, method: str = "linear", trained_length: Optional[int] = None,
                       slow: float = 1.0, fast: float = 32.0, device=None) -> Tensor:
    """Angles a position of the ``rotated / 2`` pairs, float64: ``base ** (-2 j / rotated)``, and for chains ``factor`` times as long as those that
    a network was trained on

    ``linear``: all divided by ``factor``;
    ``base``: of a greater base, ``base * factor ** (rotated / (rotated - 2))``, so that the fastest pair stays and the slowest is divided by ``factor``;
    ``bands``: pairs that turn more than ``fast`` times within ``trained_length`` stay, those that turn less than ``slow`` times are divided
    by ``factor``, and between the two the change is linear in the number of turns.  Scores then grow flatter; ``0.1 log(factor) + 1`` is the usual
    ``magnitude`` with it (:func:`rotary`)."""
    if rotated < 2 or rotated % 2:
        raise ValueError(f"an even number of channels can turn, got {rotated}")
    if not base > 0 or not factor > 0:
        raise ValueError(f"base and factor must be positive, got {base} and {factor}")
    if method == "base" and rotated > 2:
        base = base * factor ** (rotated / (rotated - 2))
    frequencies = base ** (-torch.arange(0, rotated, 2, dtype=torch.float64) / rotated)
    if method == "linear" or (method == "base" and rotated == 2):
        frequencies = frequencies / factor
    elif method == "bands":
        if trained_length is None or not 0 < slow < fast:
            raise ValueError("bands need the trained length and 0 < slow < fast")
        turns = trained_length * frequencies / (2 * math.pi)
        stays = ((turns - slow) / (fast - slow)).clamp(0, 1)
        frequencies = frequencies * stays + frequencies / factor * (1 - stays)
    elif method != "base":
        raise ValueError(f"method should be in ['linear', 'base', 'bands'], got {method}")
    return frequencies.to(device)


def rotary(q: Tensor, k: Optional[Tensor], positions: Tensor, frequencies: Tensor, num_heads: int, kv_heads: Optional[int] = None,
           interleaved: bool = False, magnitude: float = 1.0) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """``q`` and ``k`` with the channel pairs of every head turned by ``positions[node] * frequencies[pair]``, so that inner products of two nodes
    depend on how far apart they are along the chain.  All components of a node turn alike, which commutes with rotations of space.

    ``q`` is ``(N, components, channels)`` of ``num_heads`` heads, ``k`` (or ``None``: then ``q`` alone is returned) of ``kv_heads`` (as many where not given), float32
    or bfloat16, of any strides; ``positions`` (N,), int64, any values; ``frequencies`` (pairs,), float64, see :func:`rotary_frequencies`.  The
    pairs are channels ``(j, j + pairs)`` of a head, ``interleaved`` ``(2 j, 2 j + 1)``; a head's channels behind ``2 * pairs`` stay as they are.  Turned
    channels are multiplied by ``magnitude``.  Angles are formed from the exact product and reduced to one turn before float32, so far positions are as exact as near ones.

    Differentiable any number of times in ``q`` and ``k``."""
    kv_heads = num_heads if kv_heads is None else kv_heads
    _ops.check(q, k, positions, frequencies, num_heads, kv_heads)
    args = q, k, positions, frequencies, num_heads, kv_heads, bool(interleaved), float(magnitude), False
    wanted = torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad))
    out = _Rotary.apply(*args) if wanted else _ops.rotary(*args)
    return out[0] if k is None else out
