"""Rows of a table by type and the table's gradient against sums in float64."""
import pytest
import torch

from equitorch_b200 import _lib
from equitorch_b200 import nn as enn
from equitorch_b200.nn import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float64: 2.0 ** -53}


def _case(rows, types, width, dtype, skew=0.0, outside=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    prob = torch.arange(1, types + 1, dtype=torch.float64).pow(-skew)
    index = torch.multinomial(prob, rows, replacement=True, generator=g) if rows else torch.zeros(0, dtype=torch.int64)
    if outside:
        index[torch.rand(rows, generator=g) < 0.2] = -1
        index[torch.rand(rows, generator=g) < 0.1] = types
        index[torch.rand(rows, generator=g) < 0.05] = 2 ** 40
    weight = torch.randn(types, *width, generator=g).to(dtype)
    cot = torch.randn(rows, *width, generator=g).to(dtype)
    return index.to(DEV), weight.to(DEV).requires_grad_(True), cot.to(DEV)


def _check(index, weight, cot, scale):
    out = F.type_embedding(index, weight, scale)
    (gw,) = torch.autograd.grad(out, [weight], cot)
    types = weight.shape[0]
    inside = (index >= 0) & (index < types)
    at = index.clamp(0, types - 1)
    want = weight.detach().double()[at] * scale * inside.view(-1, *[1] * (weight.ndim - 1))
    eps = EPS[weight.dtype]
    # one product in the arithmetic type and one rounding of it
    assert ((out.double() - want).abs() <= 2 * eps * want.abs()).all()
    src = cot.double() * inside.view(-1, *[1] * (weight.ndim - 1))
    total = torch.zeros_like(weight, dtype=torch.float64).index_add_(0, at, src) * scale
    bulk = torch.zeros_like(total).index_add_(0, at, src.abs()) * abs(scale)
    # a sum of m terms is off by at most (m - 1) half steps of the sum of their magnitudes; the scale and the result are rounded once each
    acc = 2.0 ** -53 if weight.dtype == torch.float64 else 2.0 ** -24
    count = torch.bincount(at[inside], minlength=types).view(-1, *[1] * (weight.ndim - 1)).double()
    assert ((gw.double() - total).abs() <= count * acc * bulk + 2 * eps * (total.abs() + count * acc * bulk)).all()
    assert torch.equal(gw, torch.autograd.grad(F.type_embedding(index, weight, scale), [weight], cot)[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
@pytest.mark.parametrize("rows,types,width", [(1, 1, (1,)), (33, 119, (1, 128)), (960, 119, (128,)), (4096, 1024, (31,)), (4097, 119, (64,)),
                                              (20011, 3, (40,)), (50021, 255, (7,)), (50021, 256, (72,)), (30000, 14161, (1, 32)),
                                              (9000, 70000, (8,))])
def test_against_float64(rows, types, width, dtype):
    _check(*_case(rows, types, width, dtype, skew=0.8 if types < 20000 else 0.0), scale=0.7)


@pytest.mark.parametrize("rows,types", [(700, 20), (40000, 20), (40000, 700)])
def test_rows_of_no_type(rows, types):
    _check(*_case(rows, types, (2, 12), torch.float32, outside=True), scale=-1.5)


def test_one_type_and_rows_of_no_type_only():
    index, weight, cot = _case(30000, 5, (64,), torch.float32)
    _check(torch.full_like(index, 3), weight, cot, 1.0)
    _check(torch.full_like(index, -7), weight, cot, 1.0)


def test_long_runs_between_short_ones():
    """Runs of every length around the pieces that the sorted rows are cut into."""
    lengths = [1, 31, 32, 33, 5, 63, 64, 65, 2048, 2049, 7, 40000, 1, 96, 3, 30000]
    index, weight, cot = _case(sum(lengths), len(lengths), (24,), torch.float32)
    _check(torch.arange(len(lengths)).repeat_interleave(torch.tensor(lengths)).to(DEV), weight, cot, 1.0)


def test_empty():
    index, weight, cot = _case(0, 5, (4,), torch.float32)
    _check(index, weight, cot, 1.0)
    none = torch.zeros(0, 4, device=DEV, requires_grad=True)
    out = F.type_embedding(torch.zeros(3, dtype=torch.int64, device=DEV), none)
    assert not out.any() and out.shape == (3, 4)


def test_strided_operands_and_shapes():
    index, weight, cot = _case(6000, 11, (3, 8), torch.float32)
    wide = torch.randn(11, 3, 16, device=DEV)
    view = wide[:, :, 1::2].detach().requires_grad_(True)
    index2 = index.view(60, 100).t()
    out = F.type_embedding(index2, view, 2.0)
    assert out.shape == (100, 60, 3, 8) and torch.equal(out, 2 * view[index2])
    gout = torch.randn(100, 60, 8, 3, device=DEV).transpose(-1, -2)
    (gw,) = torch.autograd.grad(out, [view], gout)
    want = torch.zeros(11, 3, 8, dtype=torch.float64, device=DEV).index_add_(0, index2.reshape(-1), gout.double().reshape(-1, 3, 8)) * 2
    assert (gw.double() - want).abs().max() < 6000 * 2.0 ** -24 * want.abs().max()
    offset = torch.randn(11 * 24 + 1, device=DEV)[1:].view(11, 24).requires_grad_(True)          # not on a 16-byte boundary
    _check(index, offset, torch.randn(6000, 24, device=DEV), 1.0)


def test_differentiated_twice():
    index, weight, _ = _case(500, 7, (3,), torch.float64)
    assert torch.autograd.gradcheck(lambda w: F.type_embedding(index[:20], w, 1.3), [weight])
    assert torch.autograd.gradgradcheck(lambda w: F.type_embedding(index[:20], w, 1.3), [weight])


def test_captured():
    from equitorch_b200.utils.cuda_graph import GraphedStep
    index, weight, cot = _case(50000, 119, (64,), torch.float32)

    def step():
        out = F.type_embedding(index, weight, 0.5)
        return [out.detach(), *torch.autograd.grad(out, [weight], cot)]
    graphed = GraphedStep(step, DEV)
    index.copy_(torch.randint(0, 119, index.shape, device=DEV))
    got = [t.clone() for t in graphed.replay()]
    assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_other_stream():
    index, weight, cot = _case(50000, 300, (64,), torch.float32)
    want = torch.autograd.grad(F.type_embedding(index, weight), [weight], cot)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = torch.autograd.grad(F.type_embedding(index, weight), [weight], cot)[0]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_module():
    layer = enn.TypeEmbedding(10, 16, components=2, scale=0.5).to(DEV)
    types = torch.randint(0, 10, (50,), device=DEV)
    assert torch.equal(layer(types), layer.weight[types] * 0.5) and layer(types).shape == (50, 2, 16)


def test_library_refuses_missing_scratch():
    lib = _lib.lib()
    need = lib.eqt_embedding_grad_scratch(_lib.EQT_F32, 100000, 119, 64)
    assert need > 0 and lib.eqt_embedding_grad(_lib.EQT_F32, 16, 16, 16, 100000, 119, 64, 1.0, None, 0, None) == 1
    assert b"scratch" in lib.eqt_last_error()
