"""Gated linear layer against the formulas in float64, with element-wise bounds.

Each sum is off by a few float32 roundings of the sum of its terms' magnitudes (operands of float32 products are split into pairs of
TF32, 22 bits); da, du and every result are rounded to the type once."""
import math

import pytest
import torch

from equitorch_b200 import nn as enn
from equitorch_b200.nn import functional as F
from equitorch_b200.ops.fused_tp_op import check_status

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float64: 2.0 ** -53}


def _act(a, name):
    """act, its derivative and bounds of the second derivative's and the derivative's magnitude."""
    if name == "relu":
        return a.clamp(min=0), (a > 0).double()
    if name == "gelu":
        half = torch.special.ndtr(a)
        return a * half, half + a * torch.exp(-0.5 * a * a) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(a)
    return (s, s * (1 - s)) if name == "sigmoid" else (a * s, s * (1 + a * (1 - s)))


def _check(x, w, g, name):
    """|act'| <= 1.13 and |act''| <= 1 for these activations (relu: away from zero, see the caller)."""
    h = F.gated_linear(x, w, name)
    dx, dw = torch.autograd.grad(h, [x, w], g)
    check_status()
    u = U[x.dtype]
    few = 64 * 2.0 ** -53 if x.dtype == torch.float64 else 2.0 ** -19      # of a sum's magnitudes: 32 float32 roundings
    X, W, G = x.detach().double().flatten(0, -2), w.detach().double(), g.double().flatten(0, -2)
    a, v = X @ W[0], X @ W[1]
    ea, ev = few * (X.abs() @ W[0].abs()), few * (X.abs() @ W[1].abs())
    y, dy = _act(a, name)
    ey, edy = 1.13 * ea + few * (1 + a.abs()), ea + few * (1 + a.abs())
    if name == "relu":
        edy = (a.abs() <= ea).double()
    want = y * v
    tol = ey * v.abs() + y.abs() * ev + ey * ev
    assert ((h.double().flatten(0, -2) - want).abs() <= tol + u * (want.abs() + tol) + few * want.abs()).all()
    da, du = G * v * dy, G * y
    eda = G.abs() * (ev * dy.abs() + v.abs() * edy + ev * edy) + few * da.abs()
    edu = G.abs() * ey + few * du.abs()
    eda, edu = eda + u * (da.abs() + eda), edu + u * (du.abs() + edu)
    want = da @ W[0].T + du @ W[1].T
    tol = eda @ W[0].abs().T + edu @ W[1].abs().T + few * (da.abs() @ W[0].abs().T + du.abs() @ W[1].abs().T)
    assert ((dx.double().flatten(0, -2) - want).abs() <= tol + u * (want.abs() + tol) + 1e-300).all()
    for j, (d, e) in enumerate([(da, eda), (du, edu)]):
        want, tol = X.T @ d, X.abs().T @ e + few * (X.abs().T @ d.abs())
        assert ((dw[j].double() - want).abs() <= tol + u * (want.abs() + tol) + 1e-300).all()
    return h.detach(), dx, dw


def _inputs(rows, c, f, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    lead = rows if isinstance(rows, tuple) else (rows,)
    x = torch.randn(*lead, c, generator=g).to(dtype).to(DEV).requires_grad_(True)
    w = (torch.randn(2, c, f, generator=g) / math.sqrt(c)).to(dtype).to(DEV).requires_grad_(True)
    return x, w, torch.randn(*lead, f, generator=g).to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,c,f", [(1, 8, 8), (127, 64, 64), (128, 64, 128), (129, 72, 136), (960, 128, 256), (1000, 256, 200),
                                      (3001, 96, 320), (257, 16, 1024), (300, 1024, 72), (20011, 32, 40), (40000, 128, 512)])
def test_tensor_cores(rows, c, f, dtype):
    _check(*_inputs(rows, c, f, dtype), "silu")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
@pytest.mark.parametrize("rows,c,f", [(1, 1, 1), (65, 17, 33), (700, 31, 90), (3001, 7, 65), (20011, 100, 301), (300, 515, 70)])
def test_odd_sizes(rows, c, f, dtype):
    _check(*_inputs(rows, c, f, dtype), "silu")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
@pytest.mark.parametrize("name", ["silu", "gelu", "relu", "sigmoid"])
@pytest.mark.parametrize("c", [40, 37])
def test_activations(name, dtype, c):
    _check(*_inputs(300, c, 48, dtype), name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_values(dtype):
    """Projections far out on both sides of the activation."""
    x, w, g = _inputs(200, 64, 64, dtype)
    with torch.no_grad():
        x.mul_(40)
    _check(x, w, g, "silu")
    _check(x, w, g, "sigmoid")


def test_shapes_strides_and_offsets():
    x, w, g = _inputs((5, 7, 3), 32, 64, torch.float32)
    h, dx, dw = _check(x, w, g, "gelu")
    assert h.shape == (5, 7, 3, 64) and dx.shape == x.shape
    wide = torch.zeros(2, 64, 32, device=DEV)
    wide.copy_(w.detach().transpose(1, 2))
    wt = wide.transpose(1, 2).requires_grad_(True)
    xt = x.detach().permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3).requires_grad_(True)
    gt = torch.randn(5, 7, 64, 3, device=DEV).transpose(-1, -2)
    assert not wt.is_contiguous() and not xt.is_contiguous() and not gt.is_contiguous()
    _check(xt, wt, gt, "gelu")
    off = torch.randn(105 * 32 + 1, device=DEV)[1:].view(105, 32).requires_grad_(True)
    _check(off, w, g.reshape(105, 64), "gelu")
    _check(x.detach()[:1].expand(5, 7, 3, 32).requires_grad_(True), w, g, "gelu")


def test_empty():
    for rows, c, f in ((0, 8, 16), (5, 0, 16), (5, 8, 0)):
        x = torch.randn(rows, c, device=DEV, requires_grad=True)
        w = torch.randn(2, c, f, device=DEV, requires_grad=True)
        h = F.gated_linear(x, w)
        dx, dw = torch.autograd.grad(h, [x, w], torch.ones_like(h))
        assert h.shape == (rows, f) and not h.any() and not dx.any() and not dw.any()


def test_gradients_against_differences():
    for name in ("silu", "gelu", "sigmoid"):
        x, w, _ = _inputs(7, 5, 6, torch.float64)
        assert torch.autograd.gradcheck(lambda a, b: F.gated_linear(a, b, name), [x, w])


def test_one_gradient_of_two_and_same_bits_again():
    x, w, g = _inputs(5000, 64, 128, torch.bfloat16)
    h = F.gated_linear(x, w)
    dx, dw = torch.autograd.grad(h, [x, w], g, retain_graph=True)
    assert torch.equal(torch.autograd.grad(h, [x], g, retain_graph=True)[0], dx)
    assert torch.equal(torch.autograd.grad(h, [w], g)[0], dw)
    assert torch.equal(torch.autograd.grad(F.gated_linear(x, w.detach()), [x], g)[0], dx)


def test_nan_stays_in_its_row():
    x, w, g = _inputs(500, 64, 128, torch.bfloat16)
    h = F.gated_linear(x, w).detach()
    with torch.no_grad():
        x[100] = float("nan")
        x[333, 3] = float("inf")
    keep = torch.ones(500, dtype=torch.bool, device=DEV)
    keep[[100, 333]] = False
    bad = F.gated_linear(x, w)
    assert torch.equal(bad[keep], h[keep]) and bad[100].isnan().all()
    dx = torch.autograd.grad(bad, [x], g)[0]
    assert torch.isfinite(dx[keep]).all()


def test_captured_and_other_stream():
    from equitorch_b200.utils.cuda_graph import GraphedStep
    x, w, g = _inputs(5000, 64, 128, torch.float32)

    def step():
        h = F.gated_linear(x, w)
        return [h.detach(), *torch.autograd.grad(h, [x, w], g)]
    graphed, second = GraphedStep(step, DEV), GraphedStep(step, DEV)
    with torch.no_grad():
        x.copy_(torch.randn_like(x))
    want = step()
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, graphed.replay(), second.replay()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_module_and_a_block_of_all_three():
    """Types to scalars, attention within the graphs, a gated feed-forward: as they are used together, against the same in float64."""
    from equitorch_b200.graph import PackedGraphs
    gen = torch.Generator().manual_seed(2)
    sizes, c, heads = [12, 30, 1, 45], 64, 4
    n = sum(sizes)
    graphs = PackedGraphs(torch.tensor([0] + sizes).cumsum(0).to(DEV), n)
    embed = enn.TypeEmbedding(10, c, scale=0.5).to(DEV)
    attention = enn.GraphAttention(heads, cap=20.0).to(DEV)
    gate = enn.GatedLinear(c, 2 * c, "gelu").to(DEV)
    mix, down = (torch.randn(i, o, generator=gen).div(math.sqrt(i)).to(DEV).requires_grad_(True) for i, o in ((c, 3 * c), (2 * c, c)))
    types = torch.randint(0, 10, (n,), generator=gen).to(DEV)
    pos = (torch.rand(n, 3, generator=gen) * 4).to(DEV).requires_grad_(True)
    params = [embed.weight, attention.slope, gate.weight, mix, down, pos]
    x = embed(types)
    q, k, v = (x @ mix).split(c, dim=-1)
    x = x + attention(q, k, v, graphs, pos)
    out = x + gate(x) @ down
    grads = torch.autograd.grad(out.square().sum(), params)

    wide = [p.detach().double().requires_grad_(True) for p in params]
    y = wide[0][types] * 0.5
    q, k, v = ((y @ wide[3]).view(n, 3, heads, -1).permute(1, 2, 0, 3))
    s = 20 * torch.tanh(q @ k.transpose(-1, -2) * (c // heads) ** -0.5 / 20)
    diff = wide[5][:, None] - wide[5][None]
    dist = (diff.square().sum(-1) + torch.eye(n, device=DEV)).sqrt() * (1 - torch.eye(n, device=DEV))
    batch = torch.arange(len(sizes), device=DEV).repeat_interleave(torch.tensor(sizes, device=DEV))
    s = (s - wide[1][:, None, None] * dist).masked_fill(batch[:, None] != batch[None], -math.inf)
    y = y + (torch.softmax(s, -1) @ v).transpose(0, 1).reshape(n, 1, c)
    y = y + (torch.nn.functional.gelu(y @ wide[2][0]) * (y @ wide[2][1])) @ wide[4]
    want = torch.autograd.grad(y.square().sum(), wide)
    # a chain of some ten float32 sums, each within 2^-20 of its terms' magnitudes
    assert (out - y).norm() < 1e-5 * y.norm()
    assert all((a - b).norm() < 2e-5 * b.norm() for a, b in zip(grads, want))
