"""Attention of one graph so large that a sum which loses a little at every step would show it: the mean of the signed errors."""
import math

import pytest
import torch

from equitorch_b200.graph import PackedGraphs
from equitorch_b200.nn import functional as F

from .test_gpu_attention import _check, _inputs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("bias", [False, True])
def test_sums_of_one_sign(bias):
    """All queries alike, so the definition is a few sums over the nodes; values, cotangents and products of one sign."""
    n, size = 262_144, 128
    g = torch.Generator(device=DEV).manual_seed(0)
    rand = lambda *shape: torch.rand(*shape, device=DEV, generator=g)  # noqa: E731
    slant = 2 * rand(n, 1) - 1
    k = torch.randn(n, size, device=DEV, generator=g)
    k[:, :1] = slant
    q = torch.randn(1, size, device=DEV, generator=g)
    q[:, 0] = 0                                                                    # the slant is in no score
    v = (0.5 + rand(1, size)) * (1 + 0.5 * slant + 0.1 * rand(n, size))
    q, k, v, cot = (t.expand(n, size).unsqueeze(1).bfloat16().contiguous() for t in (q, k, v, 0.5 + rand(n, size)))
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    if bias:                                                                       # nodes in one place
        leaves += [torch.zeros(n, 3, device=DEV, requires_grad=True), torch.ones(1, device=DEV, requires_grad=True)]
    scale = 1 / math.sqrt(size)
    out = F.graph_attention(*leaves[:3], PackedGraphs(torch.tensor([0, n], device=DEV), n), 1, scale, None, *leaves[3:])
    dq, dk, dv = torch.autograd.grad(out, leaves[:3], cot)
    a, b, w, e = (t.detach().double()[:, 0] for t in (q, k, v, cot))
    p = torch.softmax(scale * (b @ a[0]), 0)[:, None]
    o, total = (p * w).sum(0), e.sum(0)
    far = slant.abs() > 0.2                                                        # dP - delta far from zero, of one sign for each node

    def check(name, got, want, independent):
        """A rounding to bfloat16 is off by at most 2^-8 of the value, evenly: 2^-8 / sqrt(3) in the mean square.  Of an error beside it
        that has the same sign everywhere the sums may have 1e-4 (a 40th of a rounding)."""
        error = float(((got.double() - want) / want).mean())
        assert abs(error) <= 1e-4 + 5 * 2.0 ** -8 / math.sqrt(3 * independent), f"{name}: {error:.3g} of the value in the mean"
    check("out", out.detach()[:8, 0], o.expand(8, size), size)                     # rows are alike, bit for bit
    # weights are rounded once a node, cotangents' sums once a column
    check("dv", dv[:, 0], p * total, n)
    # with positions the columns' pass goes by an exact delta, without them by that of the rounded result, off by up to 2^-8 of itself
    if bias:
        check("dk", dk[:, 0, 1:][far[:, 0]], (scale * p * ((w - o) @ total)[:, None] * a[:1, 1:])[far[:, 0]], int(far.sum()))
    check("dq", dq[:, 0, 0], scale * (e @ ((w - o).T @ (p * b[:, :1])))[:, 0], n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size,sizes", [(16, [5, 8192, 8193, 0, 8260, 33]), (64, [16385, 7]), (128, [8200])])
@pytest.mark.parametrize("bias,cap", [(True, 10.0), (False, None)])
def test_around_the_border_against_float64(dtype, size, sizes, bias, cap):
    """Sums that join another sum never, once and twice, beside small graphs."""
    leaves, cot, graphs = _inputs(sizes, 1, 1, size, dtype, bias, outside=(2, 1))
    assert graphs.tile_rows == 64 and graphs.longest == max(sizes)
    _check(leaves, cot, graphs, 1, 1.5 / math.sqrt(size), cap)


def test_scores_that_grow_along_the_keys():
    """The greatest score moves on after every join, so the waiting sums change their unit each time."""
    n = 17_000
    g = torch.Generator().manual_seed(4)
    q, k, v, cot = (torch.randn(n, 1, 32, generator=g) for _ in range(4))
    q[:, 0, 0] = torch.linspace(-1, 1, n)[torch.randperm(n, generator=g)]
    k[:, 0, 0] = torch.linspace(0, 60, n)
    leaves = [t.bfloat16().to(DEV).requires_grad_(True) for t in (q, k, v)]
    _check(leaves, cot.bfloat16().to(DEV), PackedGraphs(torch.tensor([0, n], device=DEV), n), 1, 0.7, None)
