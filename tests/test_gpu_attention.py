"""Attention within packed graphs against the formulas in float64.

Tolerances are element-wise bounds: a result is a sum of products, and each source of error is carried through it with the magnitudes
of the terms.  ``u`` is the rounding of the features' type (half a step), ``F`` a few float32 roundings."""
import math

import pytest
import torch

from equitorch_b200 import nn as enn
from equitorch_b200.graph import PackedGraphs
from equitorch_b200.nn import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FEW = 2.0 ** -20                 # 16 roundings of float32; a TF32 pair keeps 22 bits, an inner product has at most 128 terms whose
                                 # roundings add up with changing signs


def _inputs(sizes, comps, heads, size, dtype, bias, seed=0, outside=(0, 0), spread=3.0):
    g = torch.Generator().manual_seed(seed)
    n = sum(sizes) + sum(outside)
    q, k, v, cot = (torch.randn(n, comps, heads * size, generator=g).to(dtype).to(DEV) for _ in range(4))
    ptr = torch.tensor([outside[0]] + list(sizes)).cumsum(0)
    pos = (torch.rand(n, 3, generator=g) * spread).to(DEV) if bias else None
    slope = (torch.rand(heads, generator=g) + 0.2).to(DEV) if bias else None
    leaves = [t.requires_grad_(True) for t in (q, k, v, pos, slope) if t is not None]
    return leaves, cot, PackedGraphs(ptr.to(DEV), n)


def _reference(leaves, cot, graphs, heads, scale, cap):
    """Results and bounds, in float64: [out, dq, dk, dv, dpos, dslope]."""
    q, k, v = (t.detach().double() for t in leaves[:3])
    pos, slope = (t.detach().double() for t in leaves[3:]) if len(leaves) > 3 else (None, None)
    n, d, c = q.shape
    u = 2.0 ** -8 if leaves[0].dtype == torch.bfloat16 else FEW           # of a product's operand, and of a stored result
    shape = (n, d, heads, c // heads)
    val = [torch.zeros(shape, dtype=torch.float64, device=DEV) for _ in range(4)]
    tol = [torch.zeros_like(t) for t in val]
    dpos, tpos = (torch.zeros(n, 3, dtype=torch.float64, device=DEV) for _ in range(2))
    dslope, tslope = (torch.zeros(heads, dtype=torch.float64, device=DEV) for _ in range(2))
    q, k, v, g = (t.reshape(shape) for t in (q, k, v, cot.double()))
    for lo, hi in zip(graphs.ptr.tolist()[:-1], graphs.ptr.tolist()[1:]):
        if lo == hi:
            continue
        r = unit = torch.zeros((), dtype=torch.float64, device=DEV)
        if pos is not None:
            diff = pos[lo:hi, None] - pos[None, lo:hi]
            r = diff.square().sum(-1).sqrt()
            unit = diff / r.clamp(min=1e-300)[..., None]
        for h in range(heads):
            a, b, w, e = (t[lo:hi, :, h].flatten(1) for t in (q, k, v, g))
            z = scale * (a @ b.T)
            t = torch.tanh(z / cap) if cap else torch.zeros_like(z)
            s = (cap * t if cap else z) - (slope[h] * r if pos is not None else 0)
            p = torch.softmax(s, 1)
            o = p @ w
            delta = (o * e).sum(1, keepdim=True)
            dp = e @ w.T
            ds = p * (dp - delta)
            slant = scale * (1 - t * t)
            dz = ds * slant
            # absolute error of a score: the product's, the tanh's (some roundings of 1, times the cap), the distance's and the largest score's
            sigma = FEW * (scale * (a.abs() @ b.abs().T) + (cap or 0) + (slope[h] * r if pos is not None else 0) + s.abs() + 1)
            tau = 4 * sigma.amax(1, keepdim=True)                          # relative error of a weight: its score's and the sum's
            bulk = e.abs() @ w.abs().T
            fine = p * (tau * (dp.abs() + delta.abs()) + FEW * (bulk + (p * bulk).sum(1, keepdim=True)))
            coarse = fine + p * (u * (o.abs() * e.abs()).sum(1, keepdim=True))      # delta from the rounded output
            dzerr = coarse * slant + dz.abs() * u + ds.abs() * scale * FEW * (1 + (cap or 0))
            for i, (value, err) in enumerate([
                    (o, (p * (u + tau)) @ w.abs()), (dz @ b, dzerr @ b.abs()), (dz.T @ a, dzerr.T @ a.abs()),
                    (p.T @ e, (p * (u + tau)).T @ e.abs())]):
                val[i][lo:hi, :, h] = value.view(hi - lo, d, -1)
                tol[i][lo:hi, :, h] = (err + (u + FEW) * (value.abs() + err)).view(hi - lo, d, -1)
            if pos is not None:
                fine = fine + FEW * (ds.abs() + p * (dp.abs() + delta.abs()))        # the sums by P dP and P, and the distances
                dslope[h] -= (ds * r).sum()
                tslope[h] += (fine * r).sum()
                dpos[lo:hi] -= slope[h] * ((ds + ds.T)[..., None] * unit).sum(1)
                tpos[lo:hi] += slope[h] * ((fine + fine.T)[..., None] * unit.abs()).sum(1)
    val, tol = [t.view(n, d, c) for t in val], [t.view(n, d, c) for t in tol]
    return (val, tol) if pos is None else (val + [dpos, dslope], tol + [tpos, tslope])


def _run(leaves, cot, graphs, heads, scale, cap):
    out = F.graph_attention(*leaves[:3], graphs, heads, scale, cap, *leaves[3:])
    return [out.detach(), *torch.autograd.grad(out, leaves, cot)]


def _check(leaves, cot, graphs, heads, scale, cap):
    got = _run(leaves, cot, graphs, heads, scale, cap)
    want, tol = _reference(leaves, cot, graphs, heads, scale, cap)
    for name, x, y, e in zip(("out", "dq", "dk", "dv", "dpos", "dslope"), got, want, tol):
        over = ((x.double() - y).abs() - e).max() if y.numel() else torch.zeros(())
        assert over <= 1e-30, f"{name}: {float(((x.double() - y).abs() / e.clamp(min=1e-300)).max()):.3g} times its bound"
    return got


SIZES = {"one": [1], "pairs": [1, 2, 0, 1, 3], "atoms": [5, 30, 16, 17, 1, 15, 32, 0, 12], "mixed": [100, 33, 31, 64, 1, 65, 7], "long": [700, 129]}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("sizes", list(SIZES))
@pytest.mark.parametrize("comps,heads,size", [(1, 4, 32), (1, 3, 64), (9, 2, 8), (4, 1, 32)])
@pytest.mark.parametrize("bias,cap", [(True, 5.0), (False, None)])
def test_against_float64(dtype, sizes, comps, heads, size, bias, cap):
    leaves, cot, graphs = _inputs(SIZES[sizes], comps, heads, size, dtype, bias)
    _check(leaves, cot, graphs, heads, 1.5 / math.sqrt(comps * size), cap)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("comps,heads,size", [(1, 5, 1), (1, 2, 3), (3, 3, 5), (1, 1, 127), (1, 2, 100), (9, 3, 14), (16, 1, 8), (1, 7, 20)])
def test_odd_head_sizes(dtype, comps, heads, size):
    leaves, cot, graphs = _inputs([40, 3, 70], comps, heads, size, dtype, True)
    _check(leaves, cot, graphs, heads, 1 / math.sqrt(comps * size), 20.0)


@pytest.mark.parametrize("rows", [16, 32, 64])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [32, 128])
def test_every_tile(rows, dtype, size):
    sizes = {16: [16, 1, 9] * 3, 32: [32, 20, 30] * 3, 64: [64, 128, 200]}[rows]
    leaves, cot, graphs = _inputs(sizes, 1, 3, size, dtype, True)
    assert graphs.tile_rows == rows
    _check(leaves, cot, graphs, 3, 1 / math.sqrt(size), None)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_no_graph_and_neighbours_with_nan(dtype):
    leaves, cot, graphs = _inputs([20, 40, 33], 1, 2, 32, dtype, True, outside=(5, 7))
    want = _check(leaves, cot, graphs, 2, 0.2, 10.0)
    inside = torch.zeros(105, dtype=torch.bool, device=DEV)
    inside[5:98] = True
    assert all(not t[~inside].any() for t in want[:5])
    bad = torch.zeros(105, dtype=torch.bool, device=DEV)
    bad[:5] = bad[98:] = bad[25:65] = True
    with torch.no_grad():
        for i, t in enumerate([*leaves[:4], cot]):
            t[bad] = [float("nan"), float("inf"), -float("inf")][i % 3]
    got = _run(leaves, cot, graphs, 2, 0.2, 10.0)
    keep = inside & ~bad
    assert all(torch.equal(a[keep], b[keep]) for a, b in zip(got[:5], want[:5]))
    assert all(not t[~inside].any() for t in got[:4])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_scores_and_coinciding_nodes(dtype):
    leaves, cot, graphs = _inputs([50, 70], 1, 2, 32, dtype, True)
    with torch.no_grad():
        leaves[3][10:20] = leaves[3][10]
        leaves[0].mul_(30)
    _check(leaves, cot, graphs, 2, 1.0, 50.0)
    _check(leaves, cot, graphs, 2, 1.0, None)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scale,cap", [(-0.3, 4.0), (-0.3, None), (0.0, 4.0), (0.0, None), (0.2, 1e-6), (0.2, 1e-12), (0.2, 1e12), (-3.0, 0.5)])
def test_scales_and_caps(dtype, scale, cap):
    leaves, cot, graphs = _inputs([20, 70], 1, 2, 32, dtype, True)
    with torch.no_grad():
        leaves[0][3] = 0                                  # products that are zero to the last bit
    got = _run(leaves, cot, graphs, 2, scale, cap)
    want, tol = _reference(leaves, cot, graphs, 2, abs(scale), cap) if scale >= 0 else _reference(
        [-leaves[0], *leaves[1:]], cot, graphs, 2, -scale, cap)
    if scale < 0:
        want[1] = -want[1]
    assert all(((x.double() - y).abs() <= e + 1e-30).all() for x, y, e in zip(got, want, tol))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_products_far_below_the_others(dtype):
    """Nodes that the others do not see, by products of -1e25: no weight, and no gradient that is not a number."""
    leaves, cot, graphs = _inputs([40], 1, 1, 32, dtype, False)
    with torch.no_grad():
        leaves[0][:, :, 0] = 1e12
        leaves[1][:, :, 0] = 0
        leaves[1][5:9, :, 0] = -1e13
    got = _run(leaves, cot, graphs, 1, 1.0, None)
    assert all(torch.isfinite(t).all() for t in got)
    seen = torch.ones(40, dtype=torch.bool, device=DEV)
    seen[5:9] = False
    rest = [t.detach()[seen].requires_grad_(True) for t in leaves]
    few = _run([leaves[0].detach()[seen].requires_grad_(True), *rest[1:]], cot[seen], PackedGraphs(torch.tensor([0, 36], device=DEV), 36), 1, 1.0, None)
    u = 2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -18
    assert (got[0][seen].double() - few[0].double()).norm() <= u * few[0].double().norm()
    assert not got[2][5:9].any() and not got[3][5:9].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides(dtype):
    """q, k, v as slices of one tensor, a gradient that is not contiguous, and tensors off the 16-byte boundary."""
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(90, 4, 3 * 48 + 1, generator=g).to(dtype).to(DEV)
    cot = torch.randn(90, 48, 4, generator=g).to(dtype).to(DEV).transpose(1, 2)
    graphs = PackedGraphs(torch.tensor([0, 30, 90], device=DEV), 90)
    for off in (0, 1):
        leaves = [qkv[:, :, off + 48 * i: off + 48 * (i + 1)].detach().requires_grad_(True) for i in range(3)]
        assert not leaves[0].is_contiguous()
        got = _check(leaves, cot, graphs, 3, 0.1, None)
        want = _run([t.detach().contiguous().requires_grad_(True) for t in leaves], cot.contiguous(), graphs, 3, 0.1, None)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    wide = torch.randn(90, 4, 96, generator=g).to(dtype).to(DEV)
    leaves = [wide[:, :, ::2].detach().requires_grad_(True) for _ in range(3)]
    _check(leaves, cot, graphs, 3, 0.1, None)
    expanded = torch.randn(1, 4, 48, generator=g).to(dtype).to(DEV).expand(90, 4, 48).detach().requires_grad_(True)
    _check([expanded, leaves[1], leaves[2]], cot, graphs, 3, 0.1, None)


def test_gradients_against_differences():
    leaves, cot, graphs = _inputs([6, 9], 1, 2, 4, torch.float32, True)
    leaves = [t.detach().requires_grad_(True) for t in leaves]
    grads = _run(leaves, cot, graphs, 2, 0.5, 3.0)[1:]

    def value(at, step):
        moved = [t.detach().double() + (step * at[1] if i == at[0] else 0) for i, t in enumerate(leaves)]
        out = _reference(moved, cot, graphs, 2, 0.5, 3.0)[0][0]
        return float((out * cot.double()).sum())
    gen = torch.Generator().manual_seed(1)
    for i, (leaf, grad) in enumerate(zip(leaves, grads)):
        way = torch.randn(leaf.shape, generator=gen).double().to(DEV)
        slope = (value((i, way), 1e-5) - value((i, way), -1e-5)) / 2e-5
        assert abs(float((grad.double() * way).sum()) - slope) < 1e-4 * float((grad.double() * way).abs().sum())


def test_same_bits_again_and_partial_gradients():
    leaves, cot, graphs = _inputs([300, 40, 90], 1, 4, 64, torch.bfloat16, True)
    a, b = _run(leaves, cot, graphs, 4, 0.1, 20.0), _run(leaves, cot, graphs, 4, 0.1, 20.0)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    q, k, v, pos, slope = (t.detach() for t in leaves)
    v.requires_grad_(True)
    out = F.graph_attention(q, k, v, graphs, 4, 0.1, 20.0, pos, slope)
    assert torch.equal(torch.autograd.grad(out, [v], cot)[0], a[3])
    with torch.no_grad():
        assert torch.equal(F.graph_attention(q, k, v, graphs, 4, 0.1, 20.0, pos, slope), a[0])


def test_rotations_leave_the_scores():
    """Rotated features and positions give the rotated result."""
    from equitorch_b200.utils.workloads import euler_from_quaternion
    ir, gen = "0e+1o+2e", torch.Generator().manual_seed(5)
    leaves, cot, graphs = _inputs([25, 40], 9, 2, 8, torch.float32, True)
    angles = euler_from_quaternion(torch.nn.functional.normalize(torch.randn(1, 4, generator=gen, dtype=torch.float64), dim=-1))
    d = enn.WignerD(ir).to(DEV)(*(a.float().to(DEV) for a in angles))[0].detach()
    q, k, v, pos, slope = (t.detach() for t in leaves)
    turn = lambda x: torch.einsum("ij,njc->nic", d.double(), x.double()).float()  # noqa: E731
    rotation = d[1:4, 1:4].double()
    perm = torch.tensor([2, 0, 1])                      # components of a vector in the order of l = 1: y, z, x
    turned = torch.empty_like(pos)
    turned[:, perm.argsort()] = (pos[:, perm.argsort()].double() @ rotation.T).float()
    plain = F.graph_attention(q, k, v, graphs, 2, 0.2, None, pos, slope)
    got = F.graph_attention(turn(q), turn(k), turn(v), graphs, 2, 0.2, None, turned, slope)
    assert (got - turn(plain)).norm() < 1e-5 * plain.norm()


def test_captured_and_other_stream():
    from equitorch_b200.utils.cuda_graph import GraphedStep
    leaves, cot, graphs = _inputs([300, 40, 90], 1, 4, 64, torch.bfloat16, True)
    step = lambda: _run(leaves, cot, graphs, 4, 0.1, 20.0)  # noqa: E731
    graphed, second = GraphedStep(step, DEV), GraphedStep(step, DEV)
    with torch.no_grad():
        for t in leaves[:3]:
            t.copy_(torch.randn_like(t))
    want = step()
    a, b = graphed.replay(), second.replay()
    assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(want, a, b))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(want, got))


def test_no_nodes_and_no_graphs():
    for ptr, n in (([0], 0), ([0, 0, 0], 0), ([4], 4), ([2, 2], 4)):
        leaves = [torch.randn(n, 1, 8, device=DEV, requires_grad=True) for _ in range(3)]
        leaves += [torch.randn(n, 3, device=DEV, requires_grad=True), torch.ones(2, device=DEV, requires_grad=True)]
        got = _run(leaves, torch.ones(n, 1, 8, device=DEV), PackedGraphs(torch.tensor(ptr, device=DEV), n), 2, 1.0, None)
        assert all(not t.any() for t in got)


@pytest.mark.parametrize("sizes,first,behind", [([1], 0, 0), ([0, 0], 0, 0), ([], 0, 3), ([30] * 70, 0, 0), ([16, 3, 0, 5], 2, 3),
                                                ([100, 64, 1, 200, 5001, 3], 0, 9), (list(range(1500)), 1, 0)])
def test_pieces_on_the_gpu_are_those_of_the_host(sizes, first, behind):
    ptr = torch.tensor([first] + sizes).cumsum(0)
    n = int(ptr[-1]) + behind
    here, there = PackedGraphs(ptr, n), PackedGraphs(ptr.to(DEV), n)
    assert (here.tile_rows, here.covers) == (there.tile_rows, there.covers)
    assert sorted(here.tiles.tolist()) == sorted(there.tiles.tolist())
    lengths = [hi - lo for _, lo, hi, _ in there.tiles.tolist()]
    assert all(2 * a >= b for a, b in zip(lengths, lengths[1:]))               # by classes of size, the largest first
    assert torch.equal(here.to(DEV).tiles, here.tiles.to(DEV))


def test_bad_boundaries_on_the_gpu():
    for ptr, n in ([0, 5, 3], 5), ([-1, 5], 5), ([0, 6], 5), ([0, 2 ** 40], 5):
        with pytest.raises(ValueError, match="ascend"):
            PackedGraphs(torch.tensor(ptr, device=DEV), n)


def test_module_and_batch_vector():
    batch = torch.tensor([0] * 7 + [2] * 30, device=DEV)
    graphs = PackedGraphs.from_batch(batch, 4)
    assert graphs.ptr.tolist() == [0, 7, 7, 37, 37] and graphs.covers
    layer = enn.GraphAttention(4, cap=30.0).to(DEV)
    q, k, v = (torch.randn(37, 1, 64, device=DEV) for _ in range(3))
    pos = torch.randn(37, 3, device=DEV)
    out = layer(q, k, v, graphs, pos)
    assert torch.equal(out, F.graph_attention(q, k, v, graphs, 4, None, 30.0, pos, layer.slope))
    out.sum().backward()
    assert layer.slope.grad.shape == (4,)
    half = enn.GraphAttention(4).to(DEV).bfloat16()
    assert half(q.bfloat16(), k.bfloat16(), v.bfloat16(), graphs, pos).dtype == torch.bfloat16
    plain = enn.GraphAttention(4, distance_bias=False).to(DEV)
    assert torch.equal(plain(q, k, v, graphs), F.graph_attention(q, k, v, graphs, 4))
