"""Attention within windows whose sums are long: bfloat16 products add up in an adder that truncates, so a sum may not stay in it from end to end.

Values lie between two neighbours of bfloat16, so many of any 64 in a row the upper one that the weighted mean over whole sixty-fours is at least 2^-12 above the middle and
has to round up.  Weights have eight bits, so that products have sixteen and every addition to a long sum loses some.  Pieces of 8192 terms are 512 additions, or 1024
of weights in two parts, that lose at most 2^-23 of a sum that grows to two, 2^-13 together; a sum of 100,000 terms that stays in the adder loses some 2^-10."""
import math

import pytest
import torch

from equitorch_b200.graph import PackedGraphs
from equitorch_b200.nn import functional as F
from equitorch_b200.ops.fused_tp_op import check_status

from .test_gpu_window import compare, make
from .window_reference import reference, seen

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SCALES = [0.125, -0.125]                                   # tiles of 128 nodes, and of one chain
STEP, MARGIN = 2.0 ** -7, 2.0 ** -12
LOW = 199 / 256                                             # exp(-1/4) in bfloat16
THIRD = 3 * torch.tensor(1 / 3).bfloat16().item()           # what a third's rounding makes of a sum


@pytest.fixture(autouse=True)
def no_wait_gave_up():
    yield
    check_status()


def levels(size):
    return 1 + STEP * (torch.arange(size, device=DEV) * 11 % 127)


def pattern(n, heads, size, factor=None):
    """(n, heads, size), between ``levels`` and the next number: means of ``factor`` times as much round up; or (None) those where every 64th has the weight one and the
    others LOW."""
    base = levels(size).double()
    each, start = (LOW / (63 * LOW + 1), base) if factor is None else (factor / 64, factor * base)
    count = ((base + STEP / 2 + MARGIN - start) / (STEP * each)).ceil().clamp(min=0)
    rank = torch.full((64,), 64.0, device=DEV)
    rank[(torch.arange(63, device=DEV) * 27 % 64).argsort()] = torch.arange(63.0, device=DEV)
    upper = rank[torch.arange(n, device=DEV) % 64][:, None] < count
    return (levels(size) + STEP * upper)[:, None].expand(n, heads, size)


def flat(x):
    return x.reshape(x.shape[0], 1, -1).bfloat16()


def signs(n):
    """Alternating, of every place in a sixty-four as many of each."""
    j = torch.arange(n, device=DEV)
    return 1.0 - 2.0 * ((j + j // 64) % 2)


def unit(n, heads, size, by=None):
    x = torch.zeros(n, heads, size, device=DEV)
    x[:, :, 0] = 1.0 if by is None else by[:, None]
    return x


def scores(n, scale):
    """What times ``scale`` is zero at every 64th place and -1/4 at the others."""
    return torch.where(torch.arange(n, device=DEV) % 64 == 63, 0.0, -0.25 / scale)


def run(q, k, v, g, graphs, heads, *window, **kw):
    leaves = [flat(t).requires_grad_(True) for t in (q, k, v)]
    out = F.window_attention(*leaves, graphs, heads, *window, **kw)
    return [t.view(t.shape[0], -1, q.shape[2]).double() for t in (out.detach(), *torch.autograd.grad(out, leaves, flat(g)))]


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("size", [24, 64, 128])
def test_results_and_gradients_of_queries(size, scale):
    assert math.floor(math.exp(-0.25) * 256 + 0.5) == 199
    half = 65_536                                           # behind a node, itself the first of as many more
    n = 3 * half
    graphs = PackedGraphs(torch.tensor([0, n], device=DEV), n)
    q, k, values, sign = unit(n, 1, size), unit(n, 1, size, scores(n, scale)), pattern(n, 1, size), signs(n)
    want = levels(size).double() + STEP
    out, *_ = run(q, k, values, values, graphs, 1, half, half - 1, scale=scale)
    assert (out[half:2 * half] == want).all()
    k[:, :, 1:] = (values * sign[:, None, None])[:, :, 1:]
    dq = run(q, k, unit(n, 1, size, sign), unit(n, 1, size), graphs, 1, half, half - 1, scale=scale)[1]
    assert (dq[half:2 * half, :, 1:] == scale * want[1:]).all()


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("size", [24, 64, 128])
def test_gradients_of_keys_that_heads_share(size, scale):
    """The sum goes over the heads too."""
    half, heads = 3 * 4096, 8
    n = 5 * half
    graphs = PackedGraphs(torch.tensor([0, n], device=DEV), n)
    nought, one, values, sign = torch.zeros(n, heads, size, device=DEV), torch.zeros(n, 1, size, device=DEV), pattern(n, heads, size, THIRD), signs(n)
    want = heads * (levels(size).double() + STEP)
    dv = run(nought, one, one, values, graphs, heads, half, half - 1, kv_heads=1, scale=scale)[3]
    assert (dv[2 * half:3 * half] == want).all()
    dk = run(values, one, unit(n, 1, size, sign), unit(n, heads, size), graphs, heads, half, half - 1, kv_heads=1, scale=scale)[2]
    assert (dk[2 * half:3 * half] == scale * sign[2 * half:3 * half, None, None].double() * want).all()


@pytest.mark.parametrize("tile_rows", [16, 32, 64])
def test_gradients_of_keys_that_many_heads_share_in_short_chains(tile_rows):
    """Tiles of one chain, of every height."""
    length, heads, size = 384, 1024, 8
    n = 3 * length
    graphs = PackedGraphs(torch.tensor([0, length, 2 * length, n]), n)
    graphs.tile_rows = tile_rows
    graphs.tiles = graphs._tiles(n // tile_rows)
    graphs = graphs.to(DEV)
    nought, one = torch.zeros(n, heads, size, device=DEV), torch.zeros(n, 1, size, device=DEV)
    dv = run(nought, one, one, pattern(n, heads, size, THIRD), graphs, heads, length, length, kv_heads=1, scale=-1.0)[3]
    assert (dv == heads * (levels(size).double() + STEP)).all()


@pytest.mark.parametrize("scale", SCALES)
def test_gradients_of_first_nodes_that_many_heads_share(scale):
    """From queries behind their windows; the others' are zero."""
    before, sinks, heads, size = 1534, 1, 2048, 8
    far = 8 * (before + 2)
    n = before + 1 + far
    graphs = PackedGraphs(torch.tensor([0, n], device=DEV), n)
    g = torch.zeros(n, heads, size, device=DEV)
    g[before + 1:] = pattern(far, heads, size, THIRD)
    nought, one = torch.zeros(n, heads, size, device=DEV), torch.zeros(n, 1, size, device=DEV)
    dv = run(nought, one, one, g, graphs, heads, before, 0, sinks, kv_heads=1, scale=scale)[3]
    assert (dv[0] == 8 * heads * (levels(size).double() + STEP)).all()


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("size,spread", [(64, 1.0), (64, 20.0), (128, 3.0), (24, 1.0)])
def test_against_float64(size, spread, scale):
    """Chains of which one is longer than a piece, in windows that are and in windows that are not, with scores that rise behind the first piece.

    Where all weights are rounded, the greatest too, by u of themselves at most, a result is off by the sum of p_j u |v_j - out|, at most u |out| more than that of p_j u |v_j|."""
    sizes, heads = (9000, 40, 700, 1), 2
    n = sum(sizes)
    qkv, g, graphs = make(sizes, 1, heads, 1, size, torch.bfloat16, seed=size, spread=spread)
    for window in ((8500, 20, 2), (5000, 4000, 70)):
        want, bound = reference(*qkv, g, seen(sizes, n, *window), heads, 1, scale)
        bound[0] = bound[0] + 2.0 ** -8 * want[0].abs()
        out = F.window_attention(*qkv, graphs, heads, *window, kv_heads=1, scale=scale)
        compare([out.detach(), *torch.autograd.grad(out, qkv, g)], want, bound)


@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("size", [32, 64, 128])
def test_many_tiles_of_keys_that_many_heads_share(size, scale):
    """Gradients of keys in pieces of several heads each, in tiles of few and many steps one after the other: the same bits each time."""
    sizes, heads, window = [3 + (i * 37) % 60 for i in range(30)] + [1500, 2, 400], 64, (150, 30, 3)
    n = sum(sizes)
    qkv, g, graphs = make(sizes, 1, heads, 2, size, torch.bfloat16, seed=size)

    def run_it():
        out = F.window_attention(*qkv, graphs, heads, *window, kv_heads=2, scale=scale)
        return [out.detach(), *torch.autograd.grad(out, qkv, g)]
    first = run_it()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, run_it()))
    want, bound = reference(*qkv, g, seen(sizes, n, *window), heads, 2, scale)
    compare(first, want, bound)
