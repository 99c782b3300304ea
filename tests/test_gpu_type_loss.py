"""Cross entropy over types against float64, forward and backward.

Bounds: logits to within ``SUM`` of the sum of their products' absolute values (bfloat16 products are exact, sixteen at a time into a sum that truncates, at most
2^10 times 2^-23 here; of float32 six products of parts leave 2^-24, pieces of 512 terms 32 truncations); of bfloat16 the logits' gradients are rounded (``U``)."""
import pytest
import torch

from equitorch_b200.nn import functional as F
from equitorch_b200.ops.fused_tp_op import check_status

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
SUM = {torch.float32: 2.0 ** -17, torch.bfloat16: 2.0 ** -15}
TYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(autouse=True)
def no_wait_gave_up():
    yield
    check_status()


def make(n, t, c, dtype, ignored=0.2, seed=0, scale=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    x, w = (torch.randn(m, c, device=DEV, generator=gen) for m in (n, t))
    target = torch.randint(0, t, (n,), device=DEV, generator=gen)
    target[torch.rand(n, device=DEV, generator=gen) < ignored] = -1
    return x.to(dtype).requires_grad_(True), (scale * w / c ** 0.5).to(dtype).requires_grad_(True), target


def reference(x, w, target, rows):
    """Losses and gradients (of the sum of ``rows`` times the losses), and bounds of their errors."""
    dtype = x.dtype
    x, w, u, s = x.detach().double(), w.detach().double(), U[dtype], SUM[dtype]
    counts = target >= 0
    z, size = x @ w.T, x.abs() @ w.abs().T
    lse = z.logsumexp(1)
    at = target.clamp(min=0)[:, None]
    loss = torch.where(counts, lse - z.gather(1, at)[:, 0], 0.0)
    p = (z - lse[:, None]).exp()
    ez = s * size + 2.0 ** -21 * z.abs()
    elogsum = (p * ez).sum(1) + 2.0 ** -20 * (1 + lse.abs())
    eloss = torch.where(counts, elogsum + ez.gather(1, at)[:, 0] + 2.0 ** -21 * loss.abs(), 0.0)
    hot = torch.zeros_like(p).scatter_(1, at, 1.0)
    rows = torch.where(counts, rows, 0.0)[:, None]
    g = (p - hot) * rows
    eg = (p * (ez + elogsum[:, None]) * 2 + 2.0 ** -20 * (p + hot)) * rows.abs() + (u if dtype == torch.bfloat16 else 2.0 ** -22) * g.abs()
    dx, dw = g @ w, g.T @ x
    return loss, eloss, dx, (eg + s * g.abs()) @ w.abs() + u * dx.abs(), dw, (eg + s * g.abs()).T @ x.abs() + u * dw.abs()


def within(got, want, bound, what):
    over = ((got.detach().double() - want).abs() - bound).max().item() if got.numel() else 0.0
    assert over <= 1e-30 and torch.isfinite(got).all(), f"{what}: beyond its bound by {over:.3e}, of {want.abs().max().item():.3e}"


SIZES = [(1, 1, 1), (1, 2, 8), (5, 119, 16), (128, 128, 64), (129, 257, 72), (960, 119, 128), (1000, 5000, 33), (300, 14_161, 31), (7, 33_000, 100), (4000, 10, 200), (513, 777, 1000), (64, 70, 2048),
         (20_000, 300, 24)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", SIZES)
def test_against_float64(sizes, dtype):
    n, t, c = sizes
    x, w, target = make(n, t, c, dtype)
    count = (target >= 0).sum().clamp(min=1)
    loss = F.type_cross_entropy(x, w, target)
    dx, dw = torch.autograd.grad(loss, [x, w])
    want, eloss, *grads = reference(x, w, target, torch.full((n,), 1.0, dtype=torch.float64, device=DEV) / count)
    within(loss, want.sum() / count, eloss.sum() / count + 2.0 ** -22 * (want.sum() / count).abs(), "loss")
    within(dx, *grads[:2], "dx")
    within(dw, *grads[2:], "dw")
    assert not dx[target < 0].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_reductions(dtype):
    n, t, c = 200, 300, 40
    x, w, target = make(n, t, c, dtype)
    rows = torch.randn(n, device=DEV)
    each = F.type_cross_entropy(x, w, target, reduction="none")
    dx, dw = torch.autograd.grad(each, [x, w], rows)
    want, eloss, *grads = reference(x, w, target, rows.double())
    within(each, want, eloss, "losses")
    within(dx, *grads[:2], "dx")
    within(dw, *grads[2:], "dw")
    total = F.type_cross_entropy(x, w, target, reduction="sum")
    within(total, want.sum(), eloss.sum() + 2.0 ** -22 * want.sum().abs(), "sum")
    dx, dw = torch.autograd.grad(3 * total, [x, w])
    _, _, *grads = reference(x, w, target, torch.full((n,), 3.0, dtype=torch.float64, device=DEV))
    within(dx, *grads[:2], "dx")
    within(dw, *grads[2:], "dw")


@pytest.mark.parametrize("dtype", TYPES)
def test_shapes_views_and_single_gradients(dtype):
    x, w, target = make(60, 50, 24, dtype)
    loss = F.type_cross_entropy(x, w, target)
    dx, dw = torch.autograd.grad(loss, [x, w])
    again = F.type_cross_entropy(x.view(5, 12, 24), w, target.view(5, 12))
    assert torch.equal(again, loss)
    assert torch.equal(torch.autograd.grad(F.type_cross_entropy(x, w.detach(), target), x)[0], dx)
    assert torch.equal(torch.autograd.grad(F.type_cross_entropy(x.detach(), w, target), w)[0], dw)
    assert F.type_cross_entropy(x.view(5, 12, 24), w, target.view(5, 12), reduction="none").shape == (5, 12)
    wide = torch.randn(60, 60, device=DEV).to(dtype)
    for part in (wide[:, 1:25], wide.T[:, 8:32]):
        assert torch.equal(F.type_cross_entropy(part, w, target), F.type_cross_entropy(part.contiguous(), w, target))


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_do_not_count(dtype):
    """They may hold anything, and all rows may be such."""
    x, w, target = make(300, 400, 64, dtype)
    loss = F.type_cross_entropy(x, w, target)
    dx, dw = torch.autograd.grad(loss, [x, w])
    bad = x.detach().clone()
    bad[target < 0] = float("nan")
    bad[(target < 0).nonzero()[0, 0]] = float("inf")
    bad.requires_grad_(True)
    again = F.type_cross_entropy(bad, w, target)
    bx, bw = torch.autograd.grad(again, [bad, w])
    assert torch.equal(again, loss) and torch.equal(bx, dx) and torch.equal(bw, dw)
    for reduction in ("mean", "sum"):
        none = F.type_cross_entropy(x, w, torch.full_like(target, -100), reduction=reduction)
        dx, dw = torch.autograd.grad(none, [x, w])
        assert none == 0 and not dx.any() and not dw.any()


@pytest.mark.parametrize("dtype", TYPES)
def test_no_rows(dtype):
    x, w = torch.zeros(0, 8, device=DEV, dtype=dtype, requires_grad=True), torch.ones(5, 8, device=DEV, dtype=dtype, requires_grad=True)
    loss = F.type_cross_entropy(x, w, torch.zeros(0, dtype=torch.int64, device=DEV))
    dx, dw = torch.autograd.grad(loss, [x, w])
    assert loss == 0 and dx.shape == (0, 8) and not dw.any()


@pytest.mark.parametrize("dtype", TYPES)
def test_a_type_that_the_table_does_not_have(dtype):
    x, w, target = make(50, 30, 16, dtype, ignored=0.0)
    target[7] = 30
    each = F.type_cross_entropy(x, w, target, reduction="none")
    assert torch.isnan(each[7]) and torch.isfinite(each[:7]).all() and torch.isfinite(each[8:]).all()
    dx, dw = torch.autograd.grad(F.type_cross_entropy(x, w, target), [x, w])
    assert torch.isnan(dx[7]).all() and torch.isnan(dw).all() and torch.isfinite(dx[:7]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_large_and_far_logits(dtype):
    """A loss of a thousand, and rows that are sure of their type: gradients that vanish, no infinities."""
    x, w, target = make(100, 500, 64, dtype, scale=300.0)
    loss = F.type_cross_entropy(x, w, target)
    dx, dw = torch.autograd.grad(loss, [x, w])
    count = (target >= 0).sum()
    want, eloss, *grads = reference(x, w, target, torch.full((100,), 1.0, dtype=torch.float64, device=DEV) / count)
    within(loss, want.sum() / count, eloss.sum() / count + 2.0 ** -20 * want.sum() / count, "loss")
    assert torch.isfinite(dx).all() and torch.isfinite(dw).all()


def test_many_pieces_of_types():
    """Scratch for the logits' gradients holds a part of the types only."""
    n, t, c = 20_000, 20_000, 16
    x, w, target = make(n, t, c, torch.bfloat16)
    before = torch.cuda.max_memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    start = torch.cuda.memory_allocated()
    loss = F.type_cross_entropy(x, w, target)
    dx, dw = torch.autograd.grad(loss, [x, w])
    assert torch.cuda.max_memory_allocated() - start < 400 * 2 ** 20 and before >= 0
    count = (target >= 0).sum()
    rows = torch.full((n,), 1.0, dtype=torch.float64, device=DEV) / count
    want, eloss, *grads = reference(x, w, target, rows)
    within(loss, want.sum() / count, eloss.sum() / count, "loss")
    within(dx, *grads[:2], "dx")
    within(dw, *grads[2:], "dw")


def test_gradient_against_differences():
    x, w, target = make(40, 90, 16, torch.float32)
    dx, dw = torch.autograd.grad(F.type_cross_entropy(x, w, target), [x, w])
    f = lambda a, b: F.type_cross_entropy(a, b, target).double().item()  # noqa: E731
    h = 2.0 ** -6
    for i, grad in enumerate((dx, dw)):
        d = torch.randn_like(grad)
        move = lambda s: (x.detach() + s * h * d, w.detach()) if i == 0 else (x.detach(), w.detach() + s * h * d)  # noqa: E731
        one, two = (f(*move(1)) - f(*move(-1))) / (2 * h), (f(*move(2)) - f(*move(-2))) / (4 * h)
        assert abs(one - (grad.double() * d.double()).sum().item()) <= abs(two - one) + 2.0 ** -20 / h * 8


@pytest.mark.parametrize("dtype", TYPES)
def test_the_same_bits_and_replay(dtype):
    x, w, target = make(700, 3000, 64, dtype)

    def run():
        loss = F.type_cross_entropy(x, w, target)
        return [loss.detach(), *torch.autograd.grad(loss, [x, w])]

    first = run()
    assert all(torch.equal(a, b) for a, b in zip(first, run()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    with torch.no_grad():
        x.mul_(0.5)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(held, run()))


@pytest.mark.parametrize("types", [2, 3, 10, 64, 65, 119, 1000, 5000])
@pytest.mark.parametrize("spread", [1.0, 0.05])
def test_errors_as_a_whole(types, spread):
    """bfloat16.  A result's rounding leaves 1.66e-3 of its 2-norm and that of the logits' gradients as much; they are independent, so 2.35e-3 together and a
    tenth for what a thousand rows vary.  Early in training all rows' gradients are one share at the target: its rounding must not be every row's."""
    n, c = 1000, 64
    gen = torch.Generator(device=DEV).manual_seed(types)
    x, w = ((spread * torch.randn(m, c, device=DEV, generator=gen)).bfloat16().requires_grad_(True) for m in (n, types))
    target = torch.randint(types, (n,), device=DEV, generator=gen)
    got = torch.autograd.grad(F.type_cross_entropy(x, w, target), [x, w])
    xd, wd = x.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
    want = torch.autograd.grad(torch.nn.functional.cross_entropy(xd @ wd.T, target), [xd, wd])
    for what, a, b in zip(("dx", "dw"), got, want):
        error = ((a.double() - b).norm() / b.norm()).item()
        assert error < 2.6e-3, f"{what}: {error:.2e}"
