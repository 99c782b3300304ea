"""What the windows' entry points refuse besides, without a GPU."""
import ctypes as C

import torch

from equitorch_b200 import _lib


def window(**more):
    args = dict(dtype=_lib.DTYPE_CODE[torch.bfloat16], comps=1, heads=2, kv_heads=1, head_channels=8, tile_rows=64, scale=-1.0, n=40_000, num_graphs=1, longest=40_000, num_tiles=625,
                before=30_000, after=0, sinks=0, q_node=16, k_node=8, v_node=8, q=16, k=16, v=16, out=16, rest=16, stats=16, tiles=16, ptr=16, status=16, grad=16, dq=16, dk=16, dv=16)
    args = _lib.WindowAttentionArgs(**{**args, **more})
    for backward in (0, 1):
        args.scratch, args.scratch_bytes = 16, max(args.scratch_bytes, _lib.lib().eqt_window_attention_scratch(C.byref(args), backward))
    return args


def test_long_windows_of_bfloat16_need_the_highest_tiles_of_one_chain():
    """Whose kernels alone take long sums apart; a packed batch with a chain of more than 8192 nodes has these."""
    lib = _lib.lib()
    for rows in (16, 32):
        assert lib.eqt_window_attention_forward(C.byref(window(tile_rows=rows)), None) == 2
        assert lib.eqt_window_attention_backward(C.byref(window(tile_rows=rows)), None) == 2


def test_scratch_goes_by_the_nodes_and_not_by_the_chains():
    """Of first nodes' gradients: one long chain among many."""
    chains = 100_000
    n = 4000 + 20 * chains
    for sinks, groups in ((4, 1), (64, 4)):
        for dtype in (torch.float32, torch.bfloat16):
            args = window(dtype=_lib.DTYPE_CODE[dtype], n=n, num_graphs=chains + 1, longest=4000, heads=8, kv_heads=8, head_channels=64, before=30, sinks=sinks)
            size = _lib.lib().eqt_window_attention_scratch(C.byref(args), 1)
            assert size <= n * (8 + 2 * 8 * 4 + 0.55 * groups * 8 * 64) + 2 ** 20


def test_a_cache_whose_places_do_not_fit_32_bits():
    """Numbers of keys go a step beyond the capacity."""
    step = dict(dtype=0, comps=1, heads=1, kv_heads=1, head_channels=1, scale=1.0, chains=1, capacity=2 ** 31 - 1, before=2 ** 31 - 1, sinks=0, q=16, k=16, v=16, out=16, lengths=16,
                scratch=16, scratch_floats=2 ** 40)
    assert _lib.lib().eqt_window_step(C.byref(_lib.WindowStepArgs(**step)), None) == 2
