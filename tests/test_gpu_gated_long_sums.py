"""Gated products whose sums are so long that one which loses a little at every step would show it: the mean of the signed errors."""
import math

import pytest
import torch

from equitorch_b200.nn import functional as F

from .test_gpu_gated import _check, _inputs as _gated_inputs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _inputs(n, c, f):
    """Everything of one sign, projections around one."""
    g = torch.Generator(device=DEV).manual_seed(0)
    rand = lambda *shape: 0.5 + torch.rand(*shape, device=DEV, generator=g)  # noqa: E731
    return rand(n, c).bfloat16().requires_grad_(True), (rand(2, c, f) / c).bfloat16().requires_grad_(True), rand(n, f).bfloat16()


def _mean_error(got, want):
    """Against the rounded definition: sums of many terms lie closer together than the numbers of bfloat16 (65,536 terms of 0.25 to 2.25: 1 +- 0.002,
    where those are 0.004 and 0.008 apart), so their roundings do not cancel in the mean.  A shift by s of all sums moves the mean of the rounded ones by s
    times the spacing times the density of the sums where rounding changes, at most 0.4 / 0.0023 * 0.0078 = 1.35 here.  The second
    result is what chance adds where roundings differ: 2^-8 / sqrt(3) in the mean square each."""
    error = float(((got.double() - want.bfloat16().double()) / want).detach().mean())
    return error / 1.35, 5 * 2.0 ** -8 / math.sqrt(3 * want.numel())


def test_weights_of_many_rows():
    n, c, f = 200_000, 256, 9_472                                # two results' tiles an SM: nothing else asks for parts of the rows
    x, w, g = _inputs(n, c, f)
    (dw,) = torch.autograd.grad(F.gated_linear(x, w, "relu"), [w], g)
    a, u = (x.detach().double() @ w.detach()[i, :, :64].double() for i in range(2))
    for i, d in enumerate((g[:, :64].double() * u, g[:, :64].double() * a)):
        error, chance = _mean_error(dw[i, :, :64], x.detach().double().T @ d)
        # a part of 16384 rows loses 1024 times 1.8e-7, da and du are rounded evenly
        assert abs(error) <= 2e-4 + chance, f"dw[{i}]: {error:.3g}"


@pytest.mark.parametrize("c", [32_768, 65_536, 1 << 20])
def test_many_channels(c):
    n = f = 256
    x, w, g = _inputs(n, c, f)
    h = F.gated_linear(x, w, "relu")
    (dw,) = torch.autograd.grad(h, [w], g)
    a, u = (x.detach().double() @ w.detach()[i].double() for i in range(2))
    error, chance = _mean_error(h, a * u)
    # each factor is a sum of at most 32768 terms, or of pieces of 8192, which lose 9e-5 each
    lost = 3.6e-4 if c <= 32_768 else 1e-4
    assert abs(error) <= 2 * lost + chance, f"h: {error:.3g}"
    for i, d in enumerate((g.double() * u, g.double() * a)):
        error, chance = _mean_error(dw[i, :4096], x.detach()[:, :4096].double().T @ d)
        assert abs(error) <= lost + 2e-5 + chance, f"dw[{i}]: {error:.3g}"


@pytest.mark.parametrize("f", [16_384, 40_000, 1 << 20])
def test_many_hidden(f):
    n = c = 256
    x, w, g = _inputs(n, c, f)
    (dx,) = torch.autograd.grad(F.gated_linear(x, w, "relu"), [x], g)
    a, u = (x.detach().double() @ w.detach()[i].double() for i in range(2))
    W, G = w.detach().double(), g.double()
    error, chance = _mean_error(dx, (G * u) @ W[0].T + (G * a) @ W[1].T)
    # c terms lose 3e-6, two times f as above; da and du are rounded evenly
    assert abs(error) <= (3.6e-4 if 2 * f <= 32_768 else 1e-4) + 1e-5 + chance, f"dx: {error:.3g}"


@pytest.mark.parametrize("rows,c,f,name", [(130, 33_000, 70, "silu"), (129, 32_769, 136, "gelu"), (1, 70_000, 9, "sigmoid"), (300, 40_960, 512, "silu"),
                                           (257, 33_024, 64, "relu"), (70, 40, 17_001, "silu"), (300, 520, 16_392, "gelu"), (1, 8, 20_000, "silu")])
def test_long_sums_against_float64(rows, c, f, name):
    x, w, g = _gated_inputs(rows, c, f, torch.bfloat16)
    _check(x, w, g, name)
