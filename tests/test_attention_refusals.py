"""What attention within graphs refuses, and the pieces that the graphs are cut into, without a GPU."""
import ctypes

import pytest
import torch

from equitorch_b200 import _lib
from equitorch_b200 import nn as enn
from equitorch_b200.graph import PackedGraphs
from equitorch_b200.nn import functional as F


@pytest.mark.parametrize("sizes,first,behind", [([1], 0, 0), ([0, 0], 0, 0), ([30] * 7, 0, 0), ([16, 3, 0, 5], 2, 3), ([100, 64, 1, 200], 0, 9),
                                                 ([5, 1000, 2], 1, 0)])
def test_pieces_cover_every_node_once(sizes, first, behind):
    ptr = torch.tensor([first] + sizes).cumsum(0)
    n = int(ptr[-1]) + behind
    graphs = PackedGraphs(ptr, n)
    seen = torch.zeros(n, dtype=torch.int64)
    bounds = list(zip(ptr.tolist()[:-1], ptr.tolist()[1:]))
    lengths = []
    for row, lo, hi, zero in graphs.tiles.tolist():
        assert (lo, hi) in bounds and lo <= row < hi and (row - lo) % graphs.tile_rows == 0 and zero == 0
        seen[row:min(hi, row + graphs.tile_rows)] += 1
        lengths.append(hi - lo)
    assert lengths == sorted(lengths, reverse=True)
    inside = torch.zeros(n, dtype=torch.int64)
    inside[first:n - behind] = 1
    assert torch.equal(seen, inside) and graphs.covers == (first == 0 and behind == 0)


def test_bad_graphs():
    for ptr, n in ([0, 5, 3], 5), ([-1, 5], 5), ([0, 6], 5):
        with pytest.raises(ValueError, match="ascend"):
            PackedGraphs(torch.tensor(ptr), n)
    with pytest.raises(ValueError):
        PackedGraphs(torch.tensor([0, 3], dtype=torch.int32), 3)
    with pytest.raises(ValueError):
        PackedGraphs(torch.zeros(0, dtype=torch.int64), 0)
    with pytest.raises(ValueError):
        PackedGraphs(torch.tensor([0, 1]), 2 ** 31)
    for batch in ([0, 1, 0], [-1, 0], [0, 4]):
        with pytest.raises(ValueError, match="ascend"):
            PackedGraphs.from_batch(torch.tensor(batch), 4)


def test_refusals():
    graphs = PackedGraphs(torch.tensor([0, 6]), 6)
    x = torch.zeros(6, 1, 16)
    pos, slope = torch.zeros(6, 3), torch.zeros(2)
    call = lambda q=x, k=x, v=x, graphs=graphs, heads=2, **kw: F.graph_attention(q, k, v, graphs, heads, **kw)  # noqa: E731
    with pytest.raises(_lib.EqtError):
        call()
    with pytest.raises(TypeError, match="PackedGraphs"):
        call(graphs=torch.tensor([0, 6]))
    for bad in (dict(q=x[:, 0]), dict(k=x[:5]), dict(v=torch.zeros(6, 1, 8)), dict(heads=3), dict(heads=0), dict(cap=0.0), dict(cap=-1.0),
                dict(cap=float("nan")), dict(cap=float("inf")), dict(cap=1e-13), dict(scale=float("nan")),
                dict(scale=-1e13), dict(pos=pos), dict(slope=slope), dict(pos=pos[:5], slope=slope),
                dict(pos=pos, slope=torch.zeros(3))):
        with pytest.raises(ValueError):
            call(**bad)
    wide = torch.zeros(6, 9, 16)
    with pytest.raises(ValueError, match="128"):
        call(wide, wide, wide, heads=1)
    with pytest.raises(ValueError, match="nodes"):
        call(graphs=PackedGraphs(torch.tensor([0, 6]), 7))
    for bad in (dict(q=x.double(), k=x.double(), v=x.double()), dict(k=x.bfloat16()), dict(pos=pos.double(), slope=slope),
                dict(pos=pos, slope=slope.bfloat16())):
        with pytest.raises(TypeError):
            call(**bad)
    with pytest.raises(ValueError):
        enn.GraphAttention(2)(x, x, x, graphs)
    with pytest.raises(ValueError):
        enn.GraphAttention(2, distance_bias=False)(x, x, x, graphs, pos)


@pytest.mark.parametrize("wrong", [dict(dtype=1), dict(heads=0), dict(tile_rows=48), dict(cap=-1.0), dict(cap=float("nan")), dict(cap=1e20), dict(scale=float("inf")), dict(q=None),
                                   dict(tiles=None), dict(pos=16), dict(head_channels=129), dict(n=2 ** 31), dict(n=-1)])
def test_library_checks_its_arguments(wrong):
    good = dict(dtype=0, heads=2, comps=1, head_channels=8, tile_rows=16, scale=1.0, cap=0.0, n=4, num_tiles=1, tiles=16, q=16, k=16, v=16, out=16)
    lib = _lib.lib()
    assert lib.eqt_attention_forward(ctypes.byref(_lib.AttentionArgs(**{**good, **wrong})), None) in (1, 2)
    assert lib.eqt_attention_forward(None, None) == 1
    assert lib.eqt_attention_backward(ctypes.byref(_lib.AttentionArgs(**good)), None) == 1
    given = dict(grad_out=16, lse=16, dq=16, dk=16, dv=16, delta=16)
    assert lib.eqt_attention_backward(ctypes.byref(_lib.AttentionArgs(**good, **given, dpos=16, dslope=16)), None) == 1
    assert lib.eqt_pack_graphs_stats(None, 1, 16, None) == 1 and lib.eqt_pack_graphs_tiles(16, 1, 16, 1, 48, None) == 1
    assert lib.eqt_pack_graphs_tiles(16, 1, None, 1, 16, None) == 1 and lib.eqt_pack_graphs_tiles(None, 0, None, 0, 16, None) == 0
