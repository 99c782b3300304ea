"""Attention within windows of chains against float64, forward and backward."""
import pytest
import torch

from equitorch_b200.graph import PackedGraphs
from equitorch_b200.nn import functional as F

from equitorch_b200.ops.fused_tp_op import check_status

from .window_reference import reference, seen

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(autouse=True)
def no_wait_gave_up():
    yield
    check_status()


def make(sizes, comps, heads, kv_heads, size, dtype, seed=0, extra=0, spread=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    n = sum(sizes) + extra
    rand = lambda h: torch.randn(n, comps, h * size, device=DEV, generator=gen)  # noqa: E731
    q, k, v, g = (spread * rand(heads)).to(dtype), rand(kv_heads).to(dtype), rand(kv_heads).to(dtype), rand(heads).to(dtype)
    ptr = torch.tensor([0] + list(sizes), device=DEV).cumsum(0)
    return [t.requires_grad_(True) for t in (q, k, v)], g, PackedGraphs(ptr, n)


def run(qkv, g, graphs, *args, **kw):
    out = F.window_attention(*qkv, graphs, *args, **kw)
    return [out.detach(), *torch.autograd.grad(out, qkv, g)]


def compare(got, want, bound, what=("out", "dq", "dk", "dv")):
    for name, a, b, e in zip(what, got, want, bound):
        over = ((a.double() - b).abs() - e * 1.0).max().item() if a.numel() else 0.0
        assert over <= 1e-30 and torch.isfinite(a.double()).all(), f"{name}: beyond its bound by {over:.3e}, of {b.abs().max().item():.3e}"


SIZES = [(1,), (3, 0, 1, 17), (64,), (65, 127, 5), (128, 129, 1, 300)]
WINDOWS = [(0, 0, 0), (5, 0, 1), (0, 7, 2), (16, 16, 4), (64, 0, 0), (127, 3, 200), (10_000, 10_000, 0), (2 ** 31 - 1, 0, 2 ** 31 - 1)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window", WINDOWS)
@pytest.mark.parametrize("sizes", SIZES)
def test_against_float64(sizes, window, dtype):
    qkv, g, graphs = make(sizes, 1, 4, 2, 64, dtype, seed=sum(sizes))
    want, bound = reference(*qkv, g, seen(sizes, sum(sizes), *window), 4, 2, None)
    compare(run(qkv, g, graphs, 4, *window, kv_heads=2), want, bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1, 8), (1, 2, 1, 16), (4, 3, 3, 16), (9, 2, 2, 8), (1, 8, 2, 32), (1, 2, 2, 128), (4, 8, 1, 32), (1, 3, 1, 7), (3, 2, 2, 5),
                                   (1, 1, 1, 1), (1, 5, 5, 96), (2, 2, 1, 40)])
def test_heads(shape, dtype):
    comps, heads, kv_heads, size = shape
    sizes, window = (70, 2, 133), (30, 9, 3)
    qkv, g, graphs = make(sizes, comps, heads, kv_heads, size, dtype)
    want, bound = reference(*qkv, g, seen(sizes, sum(sizes), *window), heads, kv_heads, 0.3)
    compare(run(qkv, g, graphs, heads, *window, kv_heads=kv_heads, scale=0.3), want, bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("spread", [20.0, -1.0, 0.0])
def test_scores_far_apart_of_either_sign_and_zero(spread, dtype):
    sizes, window = (150, 40), (33, 2, 1)
    qkv, g, graphs = make(sizes, 1, 2, 2, 64, dtype, spread=abs(spread) or 1.0)
    scale = 0.125 if spread > 0 else -0.125 if spread else 0.0
    want, bound = reference(*qkv, g, seen(sizes, sum(sizes), *window), 2, 2, scale)
    compare(run(qkv, g, graphs, 2, *window, scale=scale), want, bound)


@pytest.mark.parametrize("dtype", TYPES)
def test_views_with_strides(dtype):
    """q, k and v as slices of one projection, components in another order in memory, an offset of one channel."""
    sizes, window, n = (90, 11), (20, 4, 2), 101
    gen = torch.Generator(device=DEV).manual_seed(3)
    for at in (0, 8, 1):                                    # whole pieces of 16 bytes, and not
        wide = torch.randn(4, n, 3 * 64 + 16, device=DEV, generator=gen).to(dtype).requires_grad_(True)
        q, k, v = (wide[:, :, at + 64 * i:at + 64 * (i + 1)].transpose(0, 1) for i in range(3))
        g = torch.randn(n, 4, 64, device=DEV, generator=gen).to(dtype)
        graphs = PackedGraphs(torch.tensor([0, 90, 101], device=DEV), n)
        out = F.window_attention(q, k, v, graphs, 4, *window)
        (grad,) = torch.autograd.grad(out, wide, g)
        want, bound = reference(q, k, v, g, seen(sizes, n, *window), 4, 4, None)
        compare([out.detach(), *(grad[:, :, at + 64 * i:at + 64 * (i + 1)].transpose(0, 1) for i in range(3))], want, bound)


@pytest.mark.parametrize("dtype", TYPES)
def test_nodes_of_no_chain(dtype):
    sizes, window = (50, 30), (8, 8, 1)
    qkv, g, _ = make(sizes, 1, 2, 1, 32, dtype, extra=20)
    graphs = PackedGraphs(torch.tensor([5, 55, 85], device=DEV), 100)
    want, bound = reference(*qkv, g, seen(sizes, 100, *window, first=5), 2, 1, None)
    got = run(qkv, g, graphs, 2, *window, kv_heads=1)
    compare(got, want, bound)
    for t in got:
        assert not t[:5].any() and not t[85:].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 2, 1, 64), (1, 1, 1, 128), (3, 2, 2, 7), (1, 4, 2, 16)])
@pytest.mark.parametrize("sinks", [1, 4, 20, 64, 65, 700])
def test_first_nodes_of_long_chains(sinks, shape, dtype):
    """Queries far behind the window of a chain's first nodes: blocks of the batch that hold several chains, one, and a part of one."""
    comps, heads, kv_heads, size = shape
    sizes, window = (3, 1500, 0, 40, 90, 2050, 700), (30, 2, sinks)
    qkv, g, _ = make(sizes, comps, heads, kv_heads, size, dtype, extra=9)
    graphs = PackedGraphs(torch.tensor([9] + list(sizes), device=DEV).cumsum(0), sum(sizes) + 9)
    want, bound = reference(*qkv, g, seen(sizes, sum(sizes) + 9, *window, first=9), heads, kv_heads, None)
    compare(run(qkv, g, graphs, heads, *window, kv_heads=kv_heads), want, bound)


@pytest.mark.parametrize("size", [64, 128])
def test_many_tiles_at_once(size):
    """Far more tiles than SMs, again and again, so that waits of every length occur: the same bits each time."""
    sizes = [50 + 450 * i // 119 for i in range(120)]
    qkv, g, graphs = make(sizes, 1, 8, 2, size, torch.bfloat16)
    first = run(qkv, g, graphs, 8, 64, 64, 4, kv_heads=2)
    for _ in range(30):
        assert all(torch.equal(a, b) for a, b in zip(first, run(qkv, g, graphs, 8, 64, 64, 4, kv_heads=2)))


@pytest.mark.parametrize("size", [64, 128, 32])
@pytest.mark.parametrize("window", [(3, 3, 0), (0, 0, 1), (40, 0, 2), (700, 0, 4), (64, 64, 300)])
def test_many_tiles_of_few_and_many_steps(window, size):
    """Thousands of tiles, of one step and of dozens, one after the other on an SM: the same bits each time, and those of the chains one by one."""
    sizes = [3 + (i * 37) % 60 for i in range(300)] + [1500, 2, 900] + [20] * 200
    qkv, g, graphs = make(sizes, 1, 8, 2, size, torch.bfloat16)
    first = run(qkv, g, graphs, 8, *window, kv_heads=2)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, run(qkv, g, graphs, 8, *window, kv_heads=2)))
    ends = torch.tensor([0] + sizes).cumsum(0).tolist()
    for c in (0, 17, 299, 300, 301, 302, 400):
        lo, hi = ends[c], ends[c + 1]
        part = [t.detach()[lo:hi].clone().requires_grad_(True) for t in qkv]
        want, bound = reference(*part, g[lo:hi], seen((hi - lo,), hi - lo, *window), 8, 2, None)
        compare([t[lo:hi] for t in first], want, bound)


def test_no_nodes():
    qkv, g, graphs = make((), 1, 2, 2, 16, torch.float32)
    assert [t.shape[0] for t in run(qkv, g, graphs, 2, 3)] == [0] * 4
    qkv, g, graphs = make((0, 0), 1, 2, 2, 16, torch.bfloat16, extra=4)
    assert not any(t.any() for t in run(qkv, g, graphs, 2, 3))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("which", [0, 1, 2, 3])
def test_what_is_not_seen_does_not_reach(which, value, dtype):
    """A value that is not finite in q, k, v or the gradient changes the rows that see it, or that it sees, and no others, by no bit."""
    sizes, (before, after, sinks), at = (150, 90), (20, 3, 2), 100
    qkv, g, graphs = make(sizes, 1, 2, 1, 64, dtype)
    mask = seen(sizes, 240, before, after, sinks).to(DEV)
    clean = run(qkv, g, graphs, 2, before, after, sinks, kv_heads=1)
    bad = [t.detach().clone() for t in (*qkv, g)]
    bad[which][at, 0, 5] = value
    got = run([t.requires_grad_(True) for t in bad[:3]], bad[3], graphs, 2, before, after, sinks, kv_heads=1)
    rows = torch.zeros(240, dtype=torch.bool, device=DEV)
    rows[at] = True
    hit = rows if which in (0, 3) else mask[:, at]          # rows whose result the value is in
    keys = mask[hit].any(0)                                 # and the keys whose gradients these are in
    hits = [hit if which != 3 else rows & False, hit, keys, keys]
    for a, b, h in zip(got, clean, hits):
        close = 4 * 2.0 ** -8 if dtype == torch.bfloat16 else 1e-4        # a row that is done again has another order of sums and no rounded weights
        assert torch.allclose(a[~h].double(), b[~h].double(), rtol=close, atol=close)
    if which == 2:
        assert (~torch.isfinite(got[0][mask[:, at]])).flatten(1).any(1).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_scores_of_minus_infinity(dtype):
    """A key whose products are all minus infinity has no weight, as if it were not seen."""
    sizes = (60,)
    qkv, g, graphs = make(sizes, 1, 1, 1, 16, dtype)
    q, k, v = (t.detach().clone() for t in qkv)
    q[:, 0, 0] = q[:, 0, 0].abs() + 0.5
    k[7, 0] = 0.0
    k[7, 0, 0] = -float("inf")
    out = F.window_attention(q, k, v, graphs, 1, 59, 59)
    keep = [i for i in range(60) if i != 7]
    s = (q.double()[:, 0] @ k.double()[keep, 0].T / 4).softmax(1)
    want = s @ v.double()[keep, 0]
    assert (out.double()[:, 0] - want).abs().max() <= (2 * 2.0 ** -8 if dtype == torch.bfloat16 else 1e-5) * v.abs().max()


def test_gradients_against_differences():
    """Of a smooth number of the result, in float32: the difference over 2 h of steps in a random direction, to its own error."""
    sizes, window = (40, 23), (6, 2, 1)
    qkv, g, graphs = make(sizes, 2, 4, 2, 8, torch.float32)
    grads = run(qkv, g, graphs, 4, *window, kv_heads=2)[1:]
    q, k, v = (t.detach() for t in qkv)
    h = 2.0 ** -6
    f = lambda *t: (F.window_attention(*t, graphs, 4, *window, kv_heads=2).double() * g.double()).sum().item()  # noqa: E731
    for i in range(3):
        d = torch.randn_like((q, k, v)[i])
        move = lambda sign: [t + (sign * h) * d if j == i else t for j, t in enumerate((q, k, v))]  # noqa: E731
        # the error of the difference is h^2 / 6 of the third derivative; a step twice as long has four times as much
        one, two = (f(*move(1)) - f(*move(-1))) / (2 * h), (f(*move(2)) - f(*move(-2))) / (4 * h)
        want = (grads[i].double() * d.double()).sum().item()
        rounding = 2.0 ** -18 * (g.abs().sum().item()) / h / 10
        assert abs(one - want) <= abs(two - one) + rounding


@pytest.mark.parametrize("dtype", TYPES)
def test_the_same_bits_and_replay(dtype):
    sizes, window = (100, 31, 200), (25, 25, 2)
    qkv, g, graphs = make(sizes, 1, 4, 2, 64, dtype)
    first = run(qkv, g, graphs, 4, *window, kv_heads=2)
    assert all(torch.equal(a, b) for a, b in zip(first, run(qkv, g, graphs, 4, *window, kv_heads=2)))
    leaves = [t.detach().clone().requires_grad_(True) for t in qkv]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(leaves, g, graphs, 4, *window, kv_heads=2)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run(leaves, g, graphs, 4, *window, kv_heads=2)
    with torch.no_grad():
        for a, b in zip(leaves, qkv):
            a.copy_(b * 0.5)
    graph.replay()
    again = run([(t.detach() * 0.5).requires_grad_(True) for t in qkv], g, graphs, 4, *window, kv_heads=2)
    assert all(torch.equal(a, b) for a, b in zip(held, again))


@pytest.mark.parametrize("dtype", TYPES)
def test_step_is_the_last_row(dtype):
    """A step over a cache is the last row of the whole chain's attention, for every length and window."""
    heads, kv_heads, size, capacity = 4, 2, 32, 300
    gen = torch.Generator(device=DEV).manual_seed(1)
    lengths = [0, 1, 2, 64, 150, 299, 300, 1000]
    keys, values = (torch.randn(len(lengths), capacity, 2, kv_heads * size, device=DEV, generator=gen).to(dtype) for _ in range(2))
    q = torch.randn(len(lengths), 2, heads * size, device=DEV, generator=gen).to(dtype)
    for before, sinks in ((0, 0), (0, 3), (10, 1), (500, 0), (100, 400)):
        got = F.window_attention_step(q, keys, values, torch.tensor(lengths, device=DEV), heads, before, sinks, kv_heads=kv_heads)
        for i, length in enumerate(lengths):
            length = min(length, capacity)
            if length == 0:
                assert not got[i].any()
                continue
            full = torch.zeros(length, 2, heads * size, device=DEV, dtype=dtype)
            full[-1] = q[i]
            (want, *_), (bound, *_) = reference(full, keys[i, :length], values[i, :length], full, seen((length,), length, before, 0, sinks), heads, kv_heads, None)
            compare([got[i]], [want[-1]], [bound[-1]], ["out"])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1, 1), (1, 8, 1, 128), (3, 6, 2, 5), (1, 7, 1, 64), (9, 4, 4, 8), (1, 3, 3, 24)])
def test_step_heads_strides_and_what_lies_behind(shape, dtype):
    comps, heads, kv_heads, size = shape
    gen = torch.Generator(device=DEV).manual_seed(2)
    cache = torch.randn(2, 40, 5, comps, kv_heads * size, device=DEV, generator=gen).to(dtype)       # nodes before chains in memory
    keys, values = cache[0].transpose(0, 1), cache[1].transpose(0, 1)
    q = torch.randn(5, comps, heads * size, device=DEV, generator=gen).to(dtype)
    lengths = [40, 17, 1, 5, 33]
    for i, length in enumerate(lengths):
        keys[i, length:] = float("nan")
        values[i, length:] = float("inf")
        keys[i, 2:max(2, length - 9)] = float("nan")        # between the first two and the window
        values[i, 2:max(2, length - 9)] = float("nan")
    got = F.window_attention_step(q, keys, values, torch.tensor(lengths, device=DEV), heads, 8, 2, kv_heads=kv_heads, scale=0.2)
    for i, length in enumerate(lengths):
        full = torch.zeros(length, comps, heads * size, device=DEV, dtype=dtype)
        full[-1] = q[i]
        (want, *_), (bound, *_) = reference(full, keys[i, :length].nan_to_num(0.0), values[i, :length].nan_to_num(0.0), full, seen((length,), length, 8, 0, 2), heads,
                                            kv_heads, 0.2)
        compare([got[i]], [want[-1]], [bound[-1]], ["out"])


def test_step_in_a_graph_while_lengths_grow():
    gen = torch.Generator(device=DEV).manual_seed(4)
    keys, values = (torch.randn(3, 600, 1, 64, device=DEV, generator=gen) for _ in range(2))
    q, lengths = torch.randn(3, 1, 64, device=DEV, generator=gen), torch.tensor([10, 200, 599], device=DEV)
    F.window_attention_step(q, keys, values, lengths, 2, 300, 2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = F.window_attention_step(q, keys, values, lengths, 2, 300, 2)
    for _ in range(3):
        graph.replay()
        assert torch.equal(held, F.window_attention_step(q, keys, values, lengths, 2, 300, 2))
        lengths += 1


@pytest.mark.parametrize("size", [32, 64, 128])
@pytest.mark.parametrize("window", [(1, 0, 0), (2, 1, 1), (30, 30, 4)])
def test_errors_of_few_and_many_nodes_as_a_whole(window, size):
    """bfloat16.  Rounding a result leaves 1.66e-3 of its 2-norm, rounding the weights (or score gradients) of a product as much of its result, so two of
    these are the most: a delta of other weights than the rows' own would be a third where few nodes are seen, and cancel."""
    sizes = (150, 3, 90, 257)
    qkv, g, graphs = make(sizes, 1, 4, 2, size, torch.bfloat16, seed=size)
    want, _ = reference(*qkv, g, seen(sizes, sum(sizes), *window), 4, 2, None)
    for what, a, b in zip(("out", "dq", "dk", "dv"), run(qkv, g, graphs, 4, *window, kv_heads=2), want):
        error = ((a.double() - b).norm() / b.norm()).item()
        assert error < 2 * 1.66e-3, f"{what}: {error:.2e}"
