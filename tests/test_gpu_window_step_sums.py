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


def test_a_long_cache():
    """bfloat16 products add up in an adder that truncates: a sum of a million keys may not stay in it.

    Of any 64 keys one has the weight one and the others exp(-1/4), 199 / 256 in bfloat16; values lie between two neighbours of bfloat16, so many of the 64 the upper one that
    the mean is at least 2^-12 above the middle and has to round up.  A warp's 8192 terms lose at most 512 times 2^-23 of a sum below two, 2^-13."""
    chains, length, size, low, step = 1200, 2 ** 20, 8, 199 / 256, 2.0 ** -7       # more chains than the GPU has places, so that none is cut for their sake
    base = 1 + step * (torch.arange(size, device=DEV) * 11 % 127)
    count = ((step / 2 + 2.0 ** -12) / (step * low / (63 * low + 1)) + 0.0 * base).ceil()
    place = torch.arange(length, device=DEV) % 64
    upper = (place * 27 % 64 - (place * 27 % 64 > 37).long())[:, None] < count      # the 64th's is 37
    values = base + step * (upper & (place != 63)[:, None])
    spread = lambda t: t.bfloat16().view(1, length, 1, size).expand(chains, -1, -1, -1)  # noqa: E731
    keys = torch.zeros(length, size, device=DEV)
    keys[:, 0] = torch.where(place == 63, 0.0, -2.0)
    q = torch.zeros(chains, 1, size, device=DEV, dtype=torch.bfloat16)
    q[:, 0, 0] = 1.0
    out = F.window_attention_step(q, spread(keys), spread(values), torch.full((chains,), length, device=DEV), 1, length, scale=0.125)
    assert (out[:, 0].double() == base.double() + step).all()
