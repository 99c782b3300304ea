"""Gated products whose sums are so long that one which loses a little at every step would show it: the mean of the signed errors."""
import math

import pytest
import torch

from equitorch_b200.nn import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _inputs(n, c, f):
    """Everything of one sign, projections around one."""
    g = torch.Generator(device=DEV).manual_seed(0)
    rand = lambda *shape: 0.5 + torch.rand(*shape, device=DEV, generator=g)  # noqa: E731
    return rand(n, c).bfloat16().requires_grad_(True), (rand(2, c, f) / c).bfloat16().requires_grad_(True), rand(n, f).bfloat16()


def _mean_error(got, want):
    """A rounding to bfloat16 is off by at most 2^-8 of the value, evenly, so 2^-8 / sqrt(3) in the mean square; `allowed` is an error of one sign."""
    error = float(((got.double() - want) / want).mean())
    return error, 5 * 2.0 ** -8 / math.sqrt(3 * want.numel())


def test_weights_of_many_rows():
    n, c, f = 200_000, 256, 9_472                                # two results' tiles an SM: nothing else asks for parts of the rows
    x, w, g = _inputs(n, c, f)
    (dw,) = torch.autograd.grad(F.gated_linear(x, w, "relu"), [w], g)
    a, u = (x.detach().double() @ w.detach()[i, :, :64].double() for i in range(2))
    for i, d in enumerate((g[:, :64].double() * u, g[:, :64].double() * a)):
        error, chance = _mean_error(dw[i, :, :64], x.detach().double().T @ d)
        # a part of 16384 rows loses 1024 times 1.8e-7, da and du are rounded evenly
        assert abs(error) <= 2e-4 + chance, f"dw[{i}]: {error:.3g}"
