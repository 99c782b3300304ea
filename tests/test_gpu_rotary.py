"""Rotary positions against float64.  A turned value is two products and a sum in float32, of a cosine and a sine within 2^-22, and a rounding to its type."""
import math

import pytest
import torch

from equitorch_b200.nn import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
TYPES = [torch.float32, torch.bfloat16]


def reference(x, positions, frequencies, heads, interleaved, magnitude, back=False):
    n, d, channels = x.shape
    half = frequencies.shape[0]
    out = x.detach().double().view(n, d, heads, channels // heads).clone()
    size = out.abs().clone()
    angle = positions.double()[:, None] * frequencies * (-1 if back else 1)
    cos, sin = (magnitude * f(angle)[:, None, None] for f in (torch.cos, torch.sin))
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    a, b = out[..., first].clone(), out[..., second].clone()
    out[..., first], out[..., second] = a * cos - b * sin, a * sin + b * cos
    size[..., first] = size[..., second] = abs(magnitude) * (a.abs() + b.abs())
    return out.view(n, d, channels), size.view(n, d, channels)


def within(got, want, size, dtype):
    over = ((got.double() - want).abs() - size * 2.0 ** -21 - want.abs() * U[dtype]).max().item() if got.numel() else 0.0
    assert over <= 0.0, f"beyond its bound by {over:.3e}"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 64, 32), (40, 1, 8, 2, 64, 32), (33, 4, 3, 1, 32, 8), (7, 1, 2, 2, 6, 3), (1000, 1, 4, 4, 20, 4), (5, 2, 12, 4, 128, 64), (100, 1, 1, 1, 16, 0),
                                   (9, 9, 2, 1, 8, 4), (3, 1, 40, 8, 128, 24), (3, 1, 1, 1, 1, 0), (17, 1, 2, 1, 1024, 512)])
def test_against_float64(shape, interleaved, dtype):
    n, comps, heads, kv_heads, size, half = shape
    gen = torch.Generator(device=DEV).manual_seed(n)
    rand = lambda h: torch.randn(n, comps, h * size, device=DEV, generator=gen).to(dtype)  # noqa: E731
    q, k, gq, gk = rand(heads), rand(kv_heads), rand(heads), rand(kv_heads)
    positions = torch.randint(-1000, 10_000_000, (n,), device=DEV, generator=gen)
    frequencies = 500.0 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / max(1, half))
    q.requires_grad_(True), k.requires_grad_(True)
    outs = F.rotary(q, k, positions, frequencies, heads, kv_heads, interleaved, 1.25)
    grads = torch.autograd.grad(outs, [q, k], [gq, gk])
    for got, x, h, back in ((outs[0], q, heads, False), (outs[1], k, kv_heads, False), (grads[0], gq, heads, True), (grads[1], gk, kv_heads, True)):
        within(got.detach(), *reference(x, positions, frequencies, h, interleaved, 1.25, back), dtype)
    with torch.no_grad():
        alone = F.rotary(q, None, positions, frequencies, heads, interleaved=interleaved, magnitude=1.25)
    assert torch.equal(alone, outs[0].detach())


@pytest.mark.parametrize("dtype", TYPES)
def test_views_of_one_projection(dtype):
    wide = torch.randn(50, 2, 3 * 64 + 8, device=DEV).to(dtype).requires_grad_(True)
    positions, frequencies = torch.arange(50, device=DEV), F.rotary_frequencies(16, device=DEV)
    for at in (0, 8, 3):
        q, k = wide[:, :, at:at + 64], wide[:, :, at + 64:at + 96]
        outs = F.rotary(q, k, positions, frequencies, 4, 2)
        same = F.rotary(q.contiguous(), k.contiguous(), positions, frequencies, 4, 2)
        assert all(torch.equal(a, b) for a, b in zip(outs, same))
        (grad,) = torch.autograd.grad(outs, wide, [torch.ones_like(t) for t in outs])
        assert not grad[:, :, :at].any() and grad[:, :, at:at + 96].any() and not grad[:, :, at + 96:].any()


def test_products_go_by_the_distance():
    """The inner product of two turned vectors is the same wherever on the chain they are."""
    q, k = (torch.randn(1, 1, 64, device=DEV, dtype=torch.float32) for _ in range(2))
    frequencies = F.rotary_frequencies(64, device=DEV)
    products = []
    for start in (0, 77, 1_000_003, 2 ** 33):
        a = F.rotary(q, None, torch.tensor([start + 5], device=DEV), frequencies, 1)
        b = F.rotary(k, None, torch.tensor([start], device=DEV), frequencies, 1)
        products.append((a.double() * b.double()).sum().item())
    bound = 64 * 2.0 ** -20 * q.abs().max().item() * k.abs().max().item()
    assert max(products) - min(products) <= bound


def test_higher_derivatives():
    q = torch.randn(6, 1, 16, device=DEV, requires_grad=True)
    positions, frequencies = torch.arange(6, device=DEV), F.rotary_frequencies(8, device=DEV)
    out = F.rotary(q, None, positions, frequencies, 1)
    (g,) = torch.autograd.grad(out.square().sum(), q, create_graph=True)
    assert torch.allclose(g, 2 * q, rtol=1e-5, atol=1e-6)    # turns keep lengths
    (h,) = torch.autograd.grad(g.sum(), q)
    assert torch.allclose(h, torch.full_like(q, 2.0), rtol=1e-5, atol=1e-6)


def test_only_one_side_wants_gradients():
    q, k = torch.randn(6, 1, 16, device=DEV, requires_grad=True), torch.randn(6, 1, 16, device=DEV)
    positions, frequencies = torch.arange(6, device=DEV), F.rotary_frequencies(16, device=DEV)
    a, b = F.rotary(q, k, positions, frequencies, 1)
    (dq,) = torch.autograd.grad((a * b).sum(), q)
    (want,) = torch.autograd.grad((F.rotary(q, None, positions, frequencies, 1) * b.detach()).sum(), q)
    assert torch.equal(dq, want)
    a, b = F.rotary(k, q, positions, frequencies, 1)
    (dk,) = torch.autograd.grad((a * b).sum(), q)
    assert torch.isfinite(dk).all()


def test_no_nodes_and_replay():
    frequencies = F.rotary_frequencies(8, device=DEV)
    assert F.rotary(torch.zeros(0, 1, 8, device=DEV), None, torch.zeros(0, dtype=torch.int64, device=DEV), frequencies, 1).shape == (0, 1, 8)
    q, positions = torch.randn(9, 1, 8, device=DEV), torch.arange(9, device=DEV)
    F.rotary(q, None, positions, frequencies, 1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = F.rotary(q, None, positions, frequencies, 1)
    positions += 1000
    graph.replay()
    assert torch.equal(held, F.rotary(q, None, positions, frequencies, 1))


def test_frequencies():
    plain = F.rotary_frequencies(64)
    assert plain.dtype == torch.float64 and plain[0] == 1 and math.isclose(plain[-1].item(), 10_000.0 ** (-62 / 64))
    assert torch.allclose(F.rotary_frequencies(64, factor=4.0), plain / 4, rtol=1e-12)
    base = F.rotary_frequencies(64, factor=4.0, method="base")
    assert base[0] == 1 and math.isclose((plain[-1] / base[-1]).item(), 4.0, rel_tol=1e-9)
    bands = F.rotary_frequencies(64, factor=4.0, method="bands", trained_length=2048)
    assert bands[0] == plain[0] and math.isclose((plain[-1] / bands[-1]).item(), 4.0, rel_tol=1e-9) and (bands <= plain).all() and (bands >= plain / 4).all()
