"""Cross entropy over types where its sums are long or nearly cancel: rows that are sure of their type, tables of many pieces, short last pieces."""
import pytest
import torch

from equitorch_b200.nn import functional as F
from equitorch_b200.ops.fused_tp_op import check_status

from .test_gpu_type_loss import SUM, TYPES, U, make, reference, within

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def no_wait_gave_up():
    yield
    check_status()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("most", [20.0, 30.0, 50.0, 100.0])
def test_rows_that_are_sure_of_their_type_early_in_the_table(most, dtype):
    """The greatest logit is among the first types and thousands follow: nothing may be lost or won on the way through them.

    A logit of the target is exact here.  Exponentials are within 2^-21 of themselves with what their arguments' rounding leaves (at most 2^-23 where they matter).  A
    thread adds 32 at a time to a sum between one and two, with a rounding of at most 2^-24 each: 4 times a tile of bfloat16, once of float32, in runs of at most 32
    tiles.  In the backward pass a weight has the log sum's rounding besides, 2^-24 of it in units of log2."""
    n, t, c, sure = 16_384, 32_768, 16, 8
    adds = (128 if dtype == torch.bfloat16 else 32) * 2.0 ** -24
    gen = torch.Generator(device=DEV).manual_seed(int(most))
    x, w = torch.randn(n, c, device=DEV, generator=gen), torch.randn(t, c, device=DEV, generator=gen) / 4
    target = torch.arange(n, device=DEV) % sure
    x[:, :sure] = 0
    x[torch.arange(n, device=DEV), target] = most + torch.arange(n, device=DEV) % 5
    w[:sure] = 0
    w[torch.arange(sure), torch.arange(sure)] = 1
    w[sure:, :sure] = 0
    x, w = x.to(dtype).requires_grad_(True), w.to(dtype).requires_grad_(True)
    losses = F.type_cross_entropy(x, w, target, reduction="none")
    dx, _ = torch.autograd.grad(losses, [x, w], torch.ones_like(losses))
    wide = w.detach().double()
    for rows in torch.arange(n, device=DEV).split(2048):
        z = x.detach()[rows].double() @ wide.T
        lse = z.logsumexp(1)
        others = z.scatter(1, target[rows][:, None], -torch.inf).logsumexp(1) - z.gather(1, target[rows][:, None])[:, 0]
        want = torch.log1p(others.exp())
        within(losses[rows], want, adds + 2.0 ** -20 * (1 + want) + want * SUM[dtype] * 8, "losses")
        p = (z - lse[:, None]).exp()
        ep = p * (2.0 ** -24 * 1.45 * lse[:, None].abs() + adds + 2.0 ** -20 + SUM[dtype] * 8)
        g = p.scatter(1, target[rows][:, None], -(others - torch.log1p(others.exp())).exp()[:, None])
        within(dx[rows], g @ wide, (ep + (U[dtype] + SUM[dtype]) * g.abs()) @ wide.abs() + U[dtype] * (g @ wide).abs(), "dx")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [30.0, 300.0])
def test_gradients_of_large_and_far_logits(scale, dtype):
    x, w, target = make(100, 500, 64, dtype, scale=scale)
    dx, dw = torch.autograd.grad(F.type_cross_entropy(x, w, target), [x, w])
    count = (target >= 0).sum()
    _, _, *grads = reference(x, w, target, torch.full((100,), 1.0, dtype=torch.float64, device=DEV) / count)
    within(dx, *grads[:2], "dx")
    within(dw, *grads[2:], "dw")


def check_against_reference(x, w, target):
    loss = F.type_cross_entropy(x, w, target)
    dx, dw = torch.autograd.grad(loss, [x, w])
    peak = torch.cuda.max_memory_allocated()
    want, eloss, *grads = reference(x, w, target, torch.full((x.shape[0],), 1.0, dtype=torch.float64, device=DEV) / (target >= 0).sum())
    within(loss, want.sum() / (target >= 0).sum(), eloss.sum() / (target >= 0).sum() + 2.0 ** -22 * want.mean(), "loss")
    within(dx, *grads[:2], "dx")
    within(dw, *grads[2:], "dw")
    assert not dx[target < 0].any()
    return peak


@pytest.mark.parametrize("dtype", TYPES)
def test_many_pieces_of_types_with_many_channels(dtype):
    """The features' gradient is one float32 sum that the pieces are added to, in scratch of the features' size and not of the table's.  A piece rounds it once, 2^-24."""
    n, t, c = (12_000, 60_000, 512) if dtype == torch.bfloat16 else (9_000, 30_000, 512)
    x, w, target = make(n, t, c, dtype)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    start, size = torch.cuda.memory_allocated(), x.element_size()
    peak = check_against_reference(x, w, target) - start
    operands = n * c * 2 if dtype == torch.bfloat16 else (n + t) * c * 6
    assert peak < 256 * 2 ** 20 + operands + n * c * 4 + (n + t) * c * size + 16 * 2 ** 20


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("more", [-1, 0, 1, 63, 64, 65, 130])
def test_short_last_pieces(more, dtype):
    """Tables that end a little before or behind a piece's end."""
    n = 20_000
    piece = (256 * 2 ** 20 // (2 if dtype == torch.bfloat16 else 6) // 20_096) // 128 * 128
    for c in (16, 20):
        check_against_reference(*make(n, piece + more, c, dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_pieces_of_few_rows_of_results(dtype):
    """Few tiles of results, so that sums over the types are cut into parts, and several pieces."""
    n, t, c = 900, (160_000 if dtype == torch.bfloat16 else 60_000), 40
    check_against_reference(*make(n, t, c, dtype))
