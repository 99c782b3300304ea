"""Rows whose offsets pass 32 bits: the last ones of tensors of more than 2^31 values."""
import pytest
import torch

from equitorch_b200.graph import PackedGraphs
from equitorch_b200.nn import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _randn(*shape, seed):
    return torch.randn(*shape, device=DEV, dtype=torch.bfloat16, generator=torch.Generator(device=DEV).manual_seed(seed))


def test_attention():
    nodes, heads, size = 281_600, 60, 128                        # 17600 graphs of 16 nodes, 2.16e9 values a tensor
    assert nodes * heads * size > 2 ** 31
    q, k, v, cot = (_randn(nodes, 1, heads * size, seed=i) for i in range(4))
    pos, slope = torch.rand(nodes, 3, device=DEV), torch.rand(heads, device=DEV)
    run = lambda a, b, c, g, p, n: (lambda leaves: (lambda out: [out.detach(), *torch.autograd.grad(out, leaves, g)])(  # noqa: E731
        F.graph_attention(*leaves[:3], PackedGraphs(torch.arange(0, n + 1, 16, device=DEV), n), heads, 0.1, 20.0, leaves[3], slope)))(
        [t.requires_grad_(True) for t in (a, b, c, p)])
    got = [t[-64:].clone() for t in run(q, k, v, cot, pos, nodes)]
    want = run(*(t.detach()[-64:].clone() for t in (q, k, v, cot, pos)), 64)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_gated():
    rows, c, f = 262_400, 16, 8_192                              # 2.15e9 values of h, twice as many of the partial gradients
    assert rows * f > 2 ** 31
    x, w = _randn(rows, c, seed=0).requires_grad_(True), (_randn(2, c, f, seed=1) / 4).requires_grad_(True)
    h = F.gated_linear(x, w)
    last = slice(rows - 300, rows)
    cot = torch.zeros(rows, f, device=DEV, dtype=torch.bfloat16)
    cot[last] = _randn(300, f, seed=2)
    dx, dw = torch.autograd.grad(h, [x, w], cot)
    wide = [t.detach().double().requires_grad_(True) for t in (x[last], w)]
    want = torch.nn.functional.silu(wide[0] @ wide[1][0]) * (wide[0] @ wide[1][1])
    grads = torch.autograd.grad(want, wide, cot[last].double())
    # one rounding of each result to bfloat16, and of the partial gradients before
    for a, b in ((h[last], want), (dx[last], grads[0]), (dw, grads[1])):
        assert (a.double() - b).norm() <= 2 * 2.0 ** -8 * b.norm()
    assert not dx[: rows - 300].any()


def test_embedding():
    rows, width = 2_100_001, 1_024
    assert rows * width > 2 ** 31
    index = torch.randint(0, 7, (rows,), device=DEV, generator=torch.Generator(device=DEV).manual_seed(0))
    weight = _randn(7, width, seed=1).requires_grad_(True)
    out = F.type_embedding(index, weight, 0.5)
    assert torch.equal(out[-1000:], weight.detach()[index[-1000:]] * 0.5)
    cot = torch.zeros_like(out)
    cot[-1000:] = _randn(1000, width, seed=2)
    (gw,) = torch.autograd.grad(out, [weight], cot)
    want = torch.zeros(7, width, device=DEV, dtype=torch.float64).index_add_(0, index[-1000:], cot[-1000:].double()) * 0.5
    assert (gw.double() - want).norm() <= 2.0 ** -8 * want.norm()
