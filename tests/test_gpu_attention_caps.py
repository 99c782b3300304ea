"""Attention with caps and scales far from one another: products of any size whose scores reach from nothing to half the cap and beyond."""
import math

import pytest
import torch

from equitorch_b200.graph import PackedGraphs
from equitorch_b200.nn import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FEW = 2.0 ** -20                 # 16 roundings of float32
TINY = 2.0 ** -126               # what float32 takes for zero here: scores 2 * 50 apart give weights of e^-100 = 4e-44, whose error is all of them


def _case(dtype, n, scale, cap, reach, seed=0):
    """q, k whose scores spread evenly over (-reach, reach) of the cap: one component of q times one of k."""
    g = torch.Generator().manual_seed(seed)
    q, k, v, cot = (torch.randn(n, 1, 32, generator=g).double() for _ in range(4))
    size = math.sqrt(reach * cap / scale)
    q, k = q * 0, k * 0
    q[:, 0, 5] = size * (0.5 + 0.5 * torch.rand(n, generator=g).double())
    k[:, 0, 5] = size * (2 * torch.rand(n, generator=g).double() - 1)
    return [t.to(dtype).to(DEV).requires_grad_(True) for t in (q, k, v)], cot.to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [15, 40, 200])                                                # tiles of 16, 32 and 64 rows
@pytest.mark.parametrize("reach", [0.01, 0.49, 3.0])                                        # the polynomial alone, and both
@pytest.mark.parametrize("cap,scale", [(30.0, 3.0), (30.0, 3e-4), (50.0, 5e-5), (20.0, 2e-7), (30.0, 3e-11), (20.0, 2e-19), (20.0, 2e-30), (4.0, 1e12)])
def test_scores_of_tens(dtype, n, reach, cap, scale):
    leaves, cot = _case(dtype, n, scale, cap, reach)
    out = F.graph_attention(*leaves, PackedGraphs(torch.tensor([0, n], device=DEV), n), 1, scale, cap)
    got = [out.detach(), *torch.autograd.grad(out, leaves, cot)]
    a, b, w, e = (t.detach().double()[:, 0] for t in (*leaves, cot))
    u = 2.0 ** -8 if dtype == torch.bfloat16 else FEW
    # the definition, and its bounds: a score is off by some roundings of itself (relative: the product, to_cap, the tanh) and of the row's largest
    z = scale * (a @ b.T)
    t = torch.tanh(z / cap)
    s = cap * t
    p = torch.softmax(s, 1)
    o, dp = p @ w, e @ w.T
    delta = (o * e).sum(1, keepdim=True)
    ds = p * (dp - delta)
    slant = scale * (1 - t * t)
    dz = ds * slant
    tau = 4 * FEW * (s.abs() + s.abs().amax(1, keepdim=True) + 1).amax(1, keepdim=True)     # relative error of a weight
    bulk = e.abs() @ w.abs().T
    err = p * (tau * (dp.abs() + delta.abs()) + FEW * (bulk + (p * bulk).sum(1, keepdim=True)) + u * ((p @ w.abs() + o.abs()) * e.abs()).sum(1, keepdim=True))
    err = err * slant + dz.abs() * u + ds.abs() * scale * FEW * 4 + TINY * scale * (1 + dp.abs() + delta.abs())
    perr = p * (u + tau) + TINY
    for name, x, want, tol in (("out", got[0], o, perr @ w.abs()), ("dq", got[1], dz @ b, err @ b.abs()), ("dk", got[2], dz.T @ a, err.T @ a.abs()),
                               ("dv", got[3], p.T @ e, perr.T @ e.abs())):
        tol = tol + (u + FEW) * (want.abs() + tol)
        over = (x.double()[:, 0] - want).abs() / tol.clamp(min=1e-300)
        assert over.max() <= 1, f"{name}: {float(over.max()):.3g} times its bound"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cap,scale", [(1e5, 0.1), (1e6, 1.0), (1e9, 1.0), (1e12, 1.0), (1e12, 1e-7), (1e12, 0.0)])
def test_large_caps_order_the_scores(dtype, cap, scale):
    """Scores of 0.1 to 0.5 of a large cap, further apart than the rounding of the greatest: each row is the value of its greatest score."""
    n = 48
    g = torch.Generator().manual_seed(1)
    place = torch.randperm(n, generator=g)
    reach = cap * (0.1 + 0.4 * place / n)                       # of a score without the cap; a 1/120 of the cap apart
    q, k, v, cot = (torch.randn(n, 1, 32, generator=g) for _ in range(4))
    q, k = q * 0, k * 0
    size = 1e12 if scale == 0 else math.sqrt(cap / scale)       # a scale of zero: products over 1.8e19, and all scores alike
    q[:, 0, 3] = size
    k[:, 0, 3] = (reach / cap).float() * size
    leaves = [t.to(dtype).to(DEV).requires_grad_(True) for t in (q, k, v)]
    out = F.graph_attention(*leaves, PackedGraphs(torch.tensor([0, n], device=DEV), n), 1, scale, cap)
    dv, = torch.autograd.grad(out, [leaves[2]], cot.to(dtype).to(DEV))
    wide, top = leaves[2].detach().double(), int(place.argmax())
    # weights are 0 or 1 to the last bit (1/48 to a few roundings for the scale of zero); a rounding of the result
    want = wide.mean(0, keepdim=True).expand_as(wide) if scale == 0 else wide[top:top + 1].expand_as(wide)
    total = cot.to(dtype).double().to(DEV).sum(0)
    u = 2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -19    # two roundings of bfloat16: weights and result
    bound = wide.abs().mean(0) if scale == 0 else want.abs()
    assert ((out.double() - want).abs() <= u * bound).all()
    bulk = cot.to(dtype).double().to(DEV).abs().sum(0)
    if scale == 0:
        assert ((dv.double() - total / n).abs() <= u * bulk / n).all()
    else:
        expect = torch.zeros_like(wide)
        expect[top] = total
        assert ((dv.double() - expect).abs() <= u * bulk).all()
