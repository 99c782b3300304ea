"""Norms of the longest rows."""
import pytest
import torch

from equitorch_b200.nn import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_a_row_of_as_many_values_as_there_may_be():
    """One channel each, so that the weight's gradient has as many."""
    gen = torch.Generator(device=DEV).manual_seed(0)
    x, g = (torch.randn(2, 2 ** 24, device=DEV, generator=gen) for _ in range(2))
    w = (1 + 0.1 * torch.randn(2 ** 24, device=DEV, generator=gen)).requires_grad_(True)
    x.requires_grad_(True)
    out, _ = F.add_rms_norm(x, None, w)
    dx, dw = torch.autograd.grad(out, [x, w], g)
    h, gw = x.detach().double(), g.double() * w.detach().double()
    r = (h.square().mean(1, keepdim=True) + 1e-6).rsqrt()
    u = h * r
    # a thread's sums have 65,536 terms, each addition within 2^-24 of the sum of absolute values: 2^-8
    assert (out.double() - u * w.double()).abs().max() <= 2.0 ** -8 * (u * w.double()).abs().max()
    assert (dw.double() - (g.double() * u).sum(0)).abs().max() <= 2.0 ** -8 * (g.double() * u).abs().max()
    want = r * (gw - u * (gw * u).mean(1, keepdim=True))
    assert (dx.double() - want).abs().max() <= 2.0 ** -8 * want.abs().max()
