"""Norms with the residual's addition against float64: forward, backward and in 8 bits.

Bounds: ``U`` half a step of the type, for each value that is rounded to it; ``C`` for what float32 arithmetic loses of sums of up to 16384 terms,
which threads take a few at a time (a sum of absolute values within 2^-18 of itself)."""
import pytest
import torch

from equitorch_b200.nn import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
C = 2.0 ** -18
TYPES = [torch.float32, torch.bfloat16]
#: rows in registers of 32, 128 and 512 threads with one to four pieces each; rows read by loops: of no whole pieces, and long ones
SHAPES = [(1, 1, 8), (5, 1, 128), (37, 4, 16), (1000, 1, 256), (3, 9, 64), (2000, 3, 128), (17, 1, 1024), (9, 1, 4096), (3, 8, 1024), (2, 1, 16384), (130, 1, 7),
          (33, 3, 5), (1, 1, 1), (7, 1, 301), (2, 2, 10_000), (600, 2, 33)]


def make(shape, dtype, residual, weight, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device=DEV, generator=gen)  # noqa: E731
    x = rand(*shape).to(dtype)
    return x, (2 * rand(*shape)).to(dtype) if residual else None, (1 + 0.3 * rand(shape[-1])).to(dtype) if weight else None, rand(*shape).to(dtype), rand(*shape).to(dtype)


def within(got, want, bound, what):
    over = ((got.double() - want).abs() - bound).max().item() if got.numel() else 0.0
    assert over <= 0.0 and torch.isfinite(got.double()).all(), f"{what}: beyond its bound by {over:.3e}, of {want.abs().max().item():.3e}"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("residual,weight", [(True, True), (False, True), (True, False), (False, False)])
@pytest.mark.parametrize("shape", SHAPES)
def test_against_float64(shape, residual, weight, dtype):
    x, res, w, g, gh = make(shape, dtype, residual, weight)
    leaves = [t.requires_grad_(True) for t in (x, res, w) if t is not None]
    out, total = F.add_rms_norm(x, res, w, 1e-3)
    grads = torch.autograd.grad([out, total], leaves, [g, gh])
    d = lambda t: t.detach().double()  # noqa: E731
    h = d(x) + (d(res) if residual else 0.0)
    wide = d(w) if weight else torch.ones(shape[-1], dtype=torch.float64, device=DEV)
    r = (h.square().mean((1, 2), keepdim=True) + 1e-3).rsqrt()
    u, gw, count = h * r, d(g) * wide, shape[1] * shape[2]
    un, sums = U[dtype], 0.0                                # the backward pass has the sum as it was before its rounding
    within(out, u * wide, (u * wide).abs() * (un + C), "out")
    within(total, h, h.abs() * un + d(x).abs() * 2.0 ** -23, "sum")
    mean, size = (gw * u).sum((1, 2), keepdim=True) / count, (gw * u).abs().sum((1, 2), keepdim=True) / count
    dx = d(gh) + r * (gw - u * mean)
    slack = r * u.abs() * (size * (2 * sums + C) + mean.abs() * sums) + C * (d(gh).abs() + r * gw.abs() + r * u.abs() * size)
    for t in grads[:1 + residual]:
        within(t, dx, slack + un * dx.abs(), "dx")
    if weight:
        dw, each = (d(g) * u).sum((0, 1)), (d(g) * u).abs().sum((0, 1))
        within(grads[-1], dw, each * (sums + C) + un * dw.abs(), "dw")


@pytest.mark.parametrize("dtype", TYPES)
def test_parts_of_the_gradient(dtype):
    """Only one of the two results is used, or only some gradients are wanted."""
    x, res, w, g, gh = make((50, 2, 64), dtype, True, True)
    leaves = [t.requires_grad_(True) for t in (x, res, w)]
    both = torch.autograd.grad(list(F.add_rms_norm(x, res, w)), leaves, [g, gh * 0])
    one = torch.autograd.grad(F.add_rms_norm(x, res, w)[0], leaves, g)
    assert all(torch.equal(a, b) for a, b in zip(both, one))
    dx, dres, dw = torch.autograd.grad(F.add_rms_norm(x, res, w)[1], leaves, gh)
    assert torch.equal(dx, gh) and torch.equal(dres, gh) and not dw.any()
    assert torch.equal(torch.autograd.grad(F.add_rms_norm(x.detach(), res.detach(), w)[0], w, g)[0], one[2])
    assert torch.equal(torch.autograd.grad(F.add_rms_norm(x.detach(), res, w.detach())[0], res, g)[0], one[1])


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_offsets(dtype):
    wide = torch.randn(30, 2, 3 * 64 + 1, device=DEV).to(dtype)
    for x in (wide[:, :, 1:65], wide[:, :, 64:128].transpose(0, 1), wide[::2, :, :64]):
        res = wide.flip(0)[:x.shape[0], :x.shape[1], :64] if x.shape[0] > 2 else None
        got, want = F.add_rms_norm(x, res), F.add_rms_norm(x.contiguous(), None if res is None else res.contiguous())
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    x = torch.randn(641, device=DEV).to(dtype)
    one = F.add_rms_norm(x[1:].view(10, 64))[0]              # no 16-byte boundary
    assert torch.allclose(one.float(), F.add_rms_norm(x[1:].clone().view(10, 64))[0].float(), rtol=2 * U[dtype], atol=1e-6)


def test_no_rows_no_channels():
    for shape in ((0, 1, 64), (0, 5), (4, 0, 8), (4, 2, 0)):
        x, w = torch.zeros(shape, device=DEV, requires_grad=True), torch.ones(shape[-1], device=DEV, requires_grad=True)
        out, total = F.add_rms_norm(x, None, w)
        dx, dw = torch.autograd.grad(out, [x, w], torch.ones_like(out))
        assert out.shape == total.shape == dx.shape == shape and not dw.any()
        values, scales, _ = F.add_rms_norm_e4m3(x.detach(), None, w.detach())
        assert values.shape == shape and scales.shape[0] == shape[0]


def nearest(t, group, count):
    """The nearest of 8 bits in float64, as the values that they stand for before the scale, and the greatest of each group."""
    cut = t.reshape(t.shape[0], count // group, group)
    most = cut.abs().amax(-1, keepdim=True)
    ratio = cut * 448.0 / torch.where(most > 0, most, torch.ones_like(most))
    grain = torch.ldexp(torch.ones_like(ratio), torch.frexp(ratio.abs()).exponent.clamp(min=-5) - 4)
    return (torch.round(ratio / grain) * grain).reshape(t.shape), most


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,group", [((40, 1, 256), None), ((40, 1, 256), 128), ((7, 4, 64), 32), ((300, 1, 2048), 128), ((9, 1, 2048), 16), ((5, 3, 40), None), ((5, 3, 40), 60),
                                         ((11, 1, 35), 5), ((2, 1, 12_000), None), ((3, 1, 384), 384), ((6, 2, 24), 1), ((4, 1, 8192), 256), ((3, 1, 16384), None)])
@pytest.mark.parametrize("residual", [True, False])
def test_eight_bits(shape, group, residual, dtype):
    """Values are the nearest to the exact quotients, to the bit; ties among them, since weights and features have few bits."""
    x, res, w, _, _ = make(shape, dtype, residual, True)
    w = (w * 4).round() / 4 if dtype == torch.bfloat16 else w
    if dtype == torch.bfloat16:
        x = (x * 8).round() / 8
    x[0] = 0
    if residual:
        res[0] = 0
    values, scales, total = F.add_rms_norm_e4m3(x, res, w, 1e-5, group)
    count = shape[1] * shape[2]
    h = x.double() + (res.double() if residual else 0.0)
    want, most = nearest(h * w.double(), group or count, count)
    assert torch.equal(values.double(), want)
    r = (h.square().mean((1, 2), keepdim=True) + 1e-5).rsqrt()
    scale = (most * r / 448.0)[..., 0]
    assert ((scales.double() - scale).abs() <= scale * C).all() and (scales[0] == 0).all()
    assert torch.equal(total, F.add_rms_norm(x, res, w, 1e-5)[1])


def test_eight_bits_of_tiny_and_huge_values():
    for size in (1e-33, 1e-38, 1e18):
        x = (torch.randn(5, 1, 64, device=DEV) * size)
        values, scales, _ = F.add_rms_norm_e4m3(x, None, None, 1e-30)
        want, _ = nearest(x.double(), 64, 64)
        assert torch.equal(values.double(), want) and torch.isfinite(scales).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_node_that_is_not_finite_keeps_to_itself(value, dtype):
    for shape in ((9, 1, 64), (9, 3, 7)):
        x, res, w, g, gh = make(shape, dtype, True, True)
        x[4, 0, 3] = value
        out, total = F.add_rms_norm(x, res, w)
        rows = [i for i in range(9) if i != 4]
        assert torch.isfinite(out[rows].float()).all() and not torch.isfinite(total[4].float()).all()
        values, scales, _ = F.add_rms_norm_e4m3(x, res, w)
        assert torch.isfinite(scales[rows]).all() and torch.isnan(scales[4]).all() and torch.isfinite(values[rows].float()).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_the_same_bits_and_replay(dtype):
    x, res, w, g, gh = make((3000, 2, 96), dtype, True, True)
    leaves = [t.requires_grad_(True) for t in (x, res, w)]

    def run():
        outs = F.add_rms_norm(x, res, w)
        return [*(o.detach() for o in outs), *torch.autograd.grad(outs, leaves, [g, gh])]

    first = run()
    assert all(torch.equal(a, b) for a, b in zip(first, run()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(first, held))


def test_rows_far_into_memory():
    """Offsets past 2^31 values."""
    n = 2 ** 31 // 4096 + 3
    x = torch.empty(n, 1, 4096, dtype=torch.bfloat16, device=DEV)
    x[:2] = 0
    x[-2:] = torch.randn(2, 1, 4096, device=DEV)
    x[2:-2] = 1
    out, _ = F.add_rms_norm(x)
    want = F.add_rms_norm(x[-2:].clone())[0]
    assert torch.equal(out[-2:], want) and (out[2:-2] == 1).all()
