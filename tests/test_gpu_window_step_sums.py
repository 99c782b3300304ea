"""A step's weights and the sum that divides them."""
import pytest
import torch

from equitorch_b200.nn import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("size", [8, 32, 64, 128])
@pytest.mark.parametrize("scale", [0.6894, 0.25, 2.0, 0.07])
def test_values_that_are_all_alike_come_out_as_they_are(scale, size):
    """bfloat16.  Whatever the weights: the sum that divides is that of the weights as they were multiplied.  exp(-0.6894) is rounded by 3.8e-3 of itself."""
    length = 700
    values = (1 + torch.arange(size, device=DEV) % 128 / 128).bfloat16().expand(2, length, 1, size)
    keys = torch.zeros(2, length, 1, size, device=DEV, dtype=torch.bfloat16)
    keys[:, torch.arange(length, device=DEV) % 8 != 7, 0, 0] = -1.0                                   # every few keys taken together hold a zero
    q = torch.zeros(2, 1, size, device=DEV, dtype=torch.bfloat16)
    q[:, 0, 0] = 1.0
    out = F.window_attention_step(q, keys, values, torch.tensor([length, 130], device=DEV), 1, length, scale=scale)
    assert torch.equal(out, values[:, 0])
