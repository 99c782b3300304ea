"""Scales of 8-bit norms tell nodes that hold, or were multiplied by, what is not finite."""
import pytest
import torch

from equitorch_b200.nn import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16]
#: rows in registers of one and of four warps, and by loops
SHAPES = [((9, 1, 64), 32), ((9, 1, 64), None), ((9, 2, 512), 128), ((9, 2, 512), None), ((9, 3, 7), 7), ((9, 3, 7), None), ((5, 1, 12_000), 100), ((9, 1, 64), 2)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,group", SHAPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf"), 1e30])
def test_a_value(value, shape, group, dtype):
    """Also one whose square float32 does not have.  All of the node's scales, no other node's."""
    x, w = torch.randn(shape, device=DEV).to(dtype), torch.ones(shape[-1], device=DEV, dtype=dtype)
    x[4, 0, 3] = value
    for res in (None, torch.randn(shape, device=DEV).to(dtype)):
        _, scales, _ = F.add_rms_norm_e4m3(x, res, w, group=group)
        assert torch.isnan(scales[4]).all() and torch.isfinite(scales[[i for i in range(shape[0]) if i != 4]]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,group", SHAPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_a_weight(value, shape, group, dtype):
    """All scales: all nodes were multiplied by it, one of zeros too."""
    x, w = torch.randn(shape, device=DEV).to(dtype), torch.ones(shape[-1], device=DEV, dtype=dtype)
    x[2] = 0
    w[5] = value
    _, scales, _ = F.add_rms_norm_e4m3(x, None, w, group=group)
    assert torch.isnan(scales).all()


def test_the_least_eps():
    """Of what float32 has below its normal numbers."""
    x = torch.zeros(3, 1, 64, device=DEV)
    out, _ = F.add_rms_norm(x, None, None, 1.5e-45)
    values, scales, _ = F.add_rms_norm_e4m3(x, None, None, 1.5e-45)
    assert not out.any() and not values.float().any() and not scales.any()
