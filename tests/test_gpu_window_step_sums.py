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
    the mean is at least 2^-12 above the middle and has to round up.  A warp's 8192 keys, in two parts of their weights, are 1024 additions that
    lose at most 2^-23 of a sum that grows to two, 2^-13 together."""
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


@pytest.mark.parametrize("size", [8, 32, 64, 128])
def test_errors_as_a_whole(size):
    """bfloat16.  Weights go into their product in two parts, which leave 2^-17 of them, so the rounding of the result is all that is to be seen: both errors are within 2^-15
    of the result's 2-norm of each other, where weights of one part leave half as much again."""
    chains, length, heads = 20, 3000, 4
    gen = torch.Generator(device=DEV).manual_seed(size)
    q, keys, values = (torch.randn(*s, device=DEV, generator=gen).bfloat16() for s in ((chains, 1, heads * size), (chains, length, 1, 2 * size), (chains, length, 1, 2 * size)))
    lengths = torch.randint(1, length + 1, (chains,), device=DEV, generator=gen)
    got = F.window_attention_step(q, keys, values, lengths, heads, 400, 3, kv_heads=2).double().view(chains, heads, size)
    for i, n in enumerate(lengths.tolist()):
        seen = torch.arange(n, device=DEV)
        seen = seen[(seen >= n - 401) | (seen < 3)]
        k, v = (t[i, seen, 0].double().view(-1, 2, 1, size).expand(-1, -1, 2, -1).reshape(-1, heads, size) for t in (keys, values))
        p = (torch.einsum("hc,jhc->hj", q[i, 0].double().view(heads, size), k) * size ** -0.5).softmax(1)
        want = torch.einsum("hj,jhc->hc", p, v)
        assert (got[i] - want).norm() <= (want.bfloat16().double() - want).norm() + 2.0 ** -15 * want.norm()
