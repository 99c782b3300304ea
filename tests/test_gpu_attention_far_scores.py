"""Attention whose scores are so large that float32 has no digits left beside them: what a row weighs, and its gradients, stay right."""
import pytest
import torch

from equitorch_b200.graph import PackedGraphs
from equitorch_b200.nn import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FEW = 2.0 ** -20                 # 16 roundings of float32


def _equal_greatest_scores(dtype, n, alike, size, capped, bias, width, scale):
    """`alike` keys have a row's greatest score, bit for bit: a weight of 1 / alike each, whose error has nothing of the score's size in it."""
    g = torch.Generator().manual_seed(n)
    k = torch.randn(1, 1, width, generator=g).expand(n, 1, width).clone()
    q, v, cot = torch.zeros(n, 1, width), *(torch.randn(n, 1, width, generator=g) for _ in range(2))
    first = torch.randperm(n, generator=g)[:alike]
    k[:, 0, 4] = -0.25
    k[first, 0, 4] = 1.0
    q[:, 0, 4] = size * (0.5 + 0.5 * torch.rand(n, generator=g))                            # the others lie at least 0.6 of the size below
    leaves = [t.to(dtype).to(DEV).requires_grad_(True) for t in (q, k, v)]
    if bias:                                                                                # nodes in one place: no distances, but all their arithmetic
        leaves += [torch.ones(n, 3, device=DEV).requires_grad_(True), torch.ones(1, device=DEV).requires_grad_(True)]
    cot, cap = cot.to(dtype).to(DEV), 4 * size if capped else None
    out = F.graph_attention(*leaves[:3], PackedGraphs(torch.tensor([0, n], device=DEV), n), 1, scale, cap, *leaves[3:])
    got = [out.detach(), *torch.autograd.grad(out, leaves, cot)]
    a, b, w, e = (t.detach().double()[:, 0] for t in (*leaves[:3], cot))
    u = 2.0 ** -8 if dtype == torch.bfloat16 else FEW
    p = torch.zeros(n, n, dtype=torch.float64, device=DEV)
    p[:, first.to(DEV)] = 1 / alike
    o, dp = p @ w, e @ w.T
    delta = (o * e).sum(1, keepdim=True)
    slant = 1 - torch.tanh(scale * (a @ b.T) / cap) ** 2 if capped else 1.0
    ds = p * (dp - delta)
    dz = ds * slant
    bulk = e.abs() @ w.abs().T
    err = p * (FEW * (dp.abs() + delta.abs() + bulk + (p * bulk).sum(1, keepdim=True)) + u * ((p @ w.abs() + o.abs()) * e.abs()).sum(1, keepdim=True))
    err = err * slant + dz.abs() * u + ds.abs() * 4 * FEW
    for name, x, want, tol in (("out", got[0], o, (p * (u + FEW)) @ w.abs()), ("dq", got[1], scale * dz @ b, scale * err @ b.abs()), ("dk", got[2], scale * dz.T @ a, scale * err.T @ a.abs()),
                               ("dv", got[3], p.T @ e, (p * (u + FEW)).T @ e.abs())):
        tol = tol + (u + FEW) * (want.abs() + tol)
        over = (x.double()[:, 0] - want).abs() / tol.clamp(min=1e-300)
        assert over.max() <= 1, f"{name}: {float(over.max()):.3g} times its bound"
    assert not bias or not (got[4].any() or got[5].any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,alike", [(15, 3), (40, 7), (200, 23)])                          # tiles of 16, 32 and 64 rows
@pytest.mark.parametrize("size", [1e3, 1e6, 1e9, 1e11])
@pytest.mark.parametrize("capped", [False, True])
@pytest.mark.parametrize("bias", [False, True])
def test_equal_greatest_scores(dtype, n, alike, size, capped, bias):
    _equal_greatest_scores(dtype, n, alike, size, capped, bias, 32, 1.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,alike", [(15, 3), (40, 7), (200, 23)])
@pytest.mark.parametrize("width", [17, 64, 72, 96, 128])                                    # every width of the kernels
@pytest.mark.parametrize("capped,bias", [(False, False), (True, False), (False, True)])
def test_equal_greatest_scores_of_other_heads(dtype, n, alike, width, capped, bias):
    """Scores that are products of a product: one rounded once more in one pass than in another would be another score."""
    _equal_greatest_scores(dtype, n, alike, 1e10, capped, bias, width, 0.7)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [15, 40, 200])
@pytest.mark.parametrize("bias", [False, True])
def test_products_of_minus_infinity(dtype, n, bias):
    """Keys whose products leave the range of the type: nobody sees them, and every gradient is what it is without them."""
    g = torch.Generator().manual_seed(2)
    q, k, v, cot = (torch.randn(n, 1, 32, generator=g) for _ in range(4))
    q[:, 0, 0], k[:, 0, 0] = 100.0, 0.0
    q[[0, n - 1], 0, 0] = 0.0                                                               # these two see them
    k[5:9, 0, 0] = -5e36                                                                    # -5e38 is past float32's -3.4e38
    leaves = [t.to(dtype).to(DEV).requires_grad_(True) for t in (q, k, v)]
    if bias:
        leaves += [torch.rand(n, 3, generator=g).to(DEV).requires_grad_(True), torch.ones(1, device=DEV).requires_grad_(True)]
    cot = cot.to(dtype).to(DEV)

    def run(leaves, cot):
        n = cot.shape[0]
        out = F.graph_attention(*leaves[:3], PackedGraphs(torch.tensor([0, n], device=DEV), n), 1, 0.5, None, *leaves[3:])
        return [out.detach(), *torch.autograd.grad(out, leaves, cot)]
    got = run(leaves, cot)
    assert all(torch.isfinite(t).all() for t in got)
    cot[0] = cot[n - 1] = 0                                                                 # and now nobody's result has anything of them
    got = run(leaves, cot)
    assert not got[2][5:9].any() and not got[3][5:9].any()
    seen = torch.ones(n, dtype=torch.bool, device=DEV)
    seen[5:9] = False
    # the same terms in tiles that begin elsewhere: roundings of sums and results, and for bfloat16 of the weights; rows 5 to 8 themselves
    # attend to the others, so gradients of k and v are compared where those rows have no cotangent
    cot[5:9] = 0
    got, few = run(leaves, cot), run([t.detach()[seen].requires_grad_(True) for t in leaves[:4]] + leaves[4:], cot[seen])
    u = 2.0 ** -6 if dtype == torch.bfloat16 else 2.0 ** -18
    got[0][[0, n - 1]], few[0][[0, -1]] = 0, 0                                              # these two see them
    for a, b in zip(got[:5], few[:5]):                                                      # of features and positions, row by row
        a = a[seen]
        assert (a.double() - b.double()).norm() <= u * b.double().norm()
