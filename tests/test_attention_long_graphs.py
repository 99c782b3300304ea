"""Which tiles a batch with a graph of more than 8192 nodes gets, and what the library asks of them, without a GPU."""
import ctypes

import pytest
import torch

from equitorch_b200 import _lib
from equitorch_b200.graph import PackedGraphs


@pytest.mark.parametrize("longest", [8191, 8192, 8193, 20000])
def test_tiles(longest):
    sizes = [3] * 4000 + [longest] + [17] * 4000
    graphs = PackedGraphs(torch.tensor([0] + sizes).cumsum(0), sum(sizes))
    assert graphs.longest == longest and graphs.tile_rows == (64 if longest > 8192 else 16)
    assert PackedGraphs(torch.tensor([0]), 7).longest == 0


def test_library_checks_the_tiles():
    good = dict(dtype=_lib.DTYPE_CODE[torch.bfloat16], heads=2, comps=1, head_channels=8, tile_rows=16, scale=1.0, n=9000, num_tiles=1, tiles=16, q=16, k=16,
                v=16, out=16)
    lib = _lib.lib()
    for wrong in (dict(longest=8193), dict(longest=0), dict(longest=8193, tile_rows=32)):
        assert lib.eqt_attention_forward(ctypes.byref(_lib.AttentionArgs(**{**good, **wrong})), None) == 2 and b"64 rows" in lib.eqt_last_error()
    assert lib.eqt_attention_forward(ctypes.byref(_lib.AttentionArgs(**good, longest=-1)), None) == 1
    assert lib.eqt_attention_forward(ctypes.byref(_lib.AttentionArgs(**{**good, "num_tiles": 0})), None) == 0
