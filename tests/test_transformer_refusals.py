"""What norms with the residual, rotary positions, attention within windows and the loss over types refuse, without a GPU."""
import ctypes as C

import pytest
import torch

from equitorch_b200 import _lib
from equitorch_b200 import nn as enn
from equitorch_b200.graph import PackedGraphs
from equitorch_b200.nn import functional as F


def test_norm():
    x, w = torch.zeros(4, 2, 8), torch.ones(8)
    for call in (F.add_rms_norm, F.add_rms_norm_e4m3):
        with pytest.raises(_lib.EqtError, match="CUDA"):
            call(x, x, w)
        with pytest.raises(ValueError, match="channels"):
            call(x[0, 0], None, w)
        with pytest.raises(ValueError, match="residual"):
            call(x, x[:3], w)
        with pytest.raises(ValueError, match="weight"):
            call(x, x, w[:7])
        with pytest.raises(TypeError, match="float32 or bfloat16"):
            call(x.double(), None, None)
        with pytest.raises(TypeError, match="residual"):
            call(x, x.bfloat16(), w)
        with pytest.raises(TypeError, match="weight"):
            call(x, x, w.bfloat16())
        for eps in (0.0, -1.0, float("nan"), float("inf")):
            with pytest.raises(ValueError, match="eps"):
                call(x, x, w, eps)
    for group in (0, -1, 3, 32):
        with pytest.raises((ValueError, _lib.EqtError), match="group|CUDA"):
            F.add_rms_norm_e4m3(x, x, w, 1e-6, group)
    with pytest.raises(ValueError, match="channels"):
        enn.AddRMSNorm(7)(x)


def test_rotary():
    q, positions, frequencies = torch.zeros(4, 1, 16), torch.zeros(4, dtype=torch.int64), F.rotary_frequencies(8)
    with pytest.raises(_lib.EqtError, match="CUDA"):
        F.rotary(q, None, positions, frequencies, 2)
    with pytest.raises(ValueError, match="heads"):
        F.rotary(q, None, positions, frequencies, 3)
    with pytest.raises(ValueError, match="does not go"):
        F.rotary(q, q[:3], positions, frequencies, 2)
    with pytest.raises(ValueError, match="does not go"):
        F.rotary(q, q, positions, frequencies, 2, 1)
    with pytest.raises(ValueError, match="pairs"):
        F.rotary(q, None, positions, F.rotary_frequencies(10), 2)
    with pytest.raises(TypeError, match="int64"):
        F.rotary(q, None, positions.int(), frequencies, 2)
    with pytest.raises(TypeError, match="float64"):
        F.rotary(q, None, positions, frequencies.float(), 2)
    with pytest.raises(ValueError, match="positions"):
        F.rotary(q, None, positions[:3], frequencies, 2)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        F.rotary(q.half(), None, positions, frequencies, 2)
    for bad in (dict(rotated=7), dict(rotated=0), dict(rotated=8, base=0.0), dict(rotated=8, factor=-1.0), dict(rotated=8, method="other"), dict(rotated=8, method="bands"),
                dict(rotated=8, method="bands", trained_length=9, slow=2.0, fast=1.0)):
        with pytest.raises(ValueError):
            F.rotary_frequencies(**bad)


def test_window():
    q, graphs = torch.zeros(6, 1, 16), PackedGraphs(torch.tensor([0, 6]), 6)
    with pytest.raises(_lib.EqtError, match="CUDA"):
        F.window_attention(q, q, q, graphs, 2, 3)
    with pytest.raises(TypeError, match="PackedGraphs"):
        F.window_attention(q, q, q, torch.tensor([0, 6]), 2, 3)
    with pytest.raises(ValueError, match="nodes"):
        F.window_attention(q[:5], q[:5], q[:5], graphs, 2, 3)
    with pytest.raises(ValueError, match="same shape"):
        F.window_attention(q, q, q[:, :, :8], graphs, 2, 3)
    with pytest.raises(ValueError, match="go together"):
        F.window_attention(q, q, q, graphs, 2, 3, kv_heads=1)
    with pytest.raises(ValueError, match="share"):
        F.window_attention(q, q, q, graphs, 2, 3, kv_heads=3)
    with pytest.raises(ValueError, match="at most 128"):
        F.window_attention(*[torch.zeros(6, 3, 88)] * 3, graphs, 2, 3)
    for window in ((-1, 0, 0), (3, -1, 0), (3, 0, -2), (2 ** 31, 0, 0), (1.5, 0, 0)):
        with pytest.raises(ValueError, match="windows"):
            F.window_attention(q, q, q, graphs, 2, *window)
    with pytest.raises(ValueError, match="scale"):
        F.window_attention(q, q, q, graphs, 2, 3, scale=float("nan"))
    with pytest.raises(TypeError, match="one type"):
        F.window_attention(q, q.bfloat16(), q, graphs, 2, 3)


def test_step():
    q, cache, lengths = torch.zeros(3, 1, 16), torch.zeros(3, 9, 1, 8), torch.ones(3, dtype=torch.int64)
    with pytest.raises(_lib.EqtError, match="CUDA"):
        F.window_attention_step(q, cache, cache, lengths, 2, 3, kv_heads=1)
    with pytest.raises(ValueError, match="cache"):
        F.window_attention_step(q, cache[0], cache[0], lengths, 2, 3, kv_heads=1)
    with pytest.raises(ValueError, match="chains"):
        F.window_attention_step(q[:2], cache, cache, lengths, 2, 3, kv_heads=1)
    with pytest.raises(ValueError, match="lengths"):
        F.window_attention_step(q, cache, cache, lengths[:2], 2, 3, kv_heads=1)
    with pytest.raises(TypeError, match="int64"):
        F.window_attention_step(q, cache, cache, lengths.int(), 2, 3, kv_heads=1)


def test_loss():
    x, w, target = torch.zeros(4, 8), torch.zeros(5, 8), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(_lib.EqtError, match="CUDA"):
        F.type_cross_entropy(x, w, target)
    with pytest.raises(ValueError, match="reduction"):
        F.type_cross_entropy(x, w, target, reduction="batchmean")
    with pytest.raises(ValueError, match="types, channels"):
        F.type_cross_entropy(x, w[0], target)
    with pytest.raises(ValueError, match="type for each row"):
        F.type_cross_entropy(x, w, target[:3])
    with pytest.raises(ValueError, match="type for each row"):
        F.type_cross_entropy(x[:, :7], w, target)
    with pytest.raises(TypeError, match="one type"):
        F.type_cross_entropy(x, w.bfloat16(), target)
    with pytest.raises(TypeError, match="int64"):
        F.type_cross_entropy(x, w, target.int())


def test_library_checks_its_arguments():
    """Before anything is launched: the addresses are none."""
    lib = _lib.lib()
    assert lib.eqt_add_rms_norm_forward(7, 16, 16, 16, 16, 16, 16, 1, 1, 8, 1e-6, None) == 1
    assert lib.eqt_add_rms_norm_forward(0, None, 16, 16, 16, 16, 16, 1, 1, 8, 1e-6, None) == 1
    assert lib.eqt_add_rms_norm_forward(0, 16, 16, 16, 16, 16, 16, -1, 1, 8, 1e-6, None) == 1
    assert lib.eqt_add_rms_norm_forward(0, 16, 16, 16, 16, 16, 16, 1, 2 ** 20, 2 ** 20, 1e-6, None) == 2
    assert lib.eqt_add_rms_norm_e4m3(0, 16, 16, 16, 16, 16, 16, 1, 1, 8, 3, 1e-6, None) == 1
    assert lib.eqt_add_rms_norm_backward(0, 16, 16, 16, 16, 16, 16, 16, 16, None, 0, 1, 1, 8, None) == 1
    assert lib.eqt_rotary(None, None) == 1 and lib.eqt_window_step(None, None) == 1
    rotary = dict(dtype=0, comps=1, heads=1, kv_heads=1, size=8, half=4, n=1, q=16, q_out=16, positions=16, frequencies=16)
    for bad, code in ((dict(dtype=9), 1), (dict(half=5), 1), (dict(size=0), 1), (dict(n=-1), 1), (dict(positions=None), 1), (dict(k=16), 1), (dict(half=600, size=1200), 2)):
        assert lib.eqt_rotary(C.byref(_lib.RotaryArgs(**{**rotary, **bad})), None) == code
    step = dict(dtype=0, comps=1, heads=2, kv_heads=1, head_channels=8, scale=1.0, chains=1, capacity=4, before=1, sinks=0, q=16, k=16, v=16, out=16, lengths=16)
    for bad, code in ((dict(heads=3, kv_heads=2), 1), (dict(before=-1), 1), (dict(lengths=None), 1), (dict(head_channels=129), 2), (dict(chains=70_000), 2)):
        assert lib.eqt_window_step(C.byref(_lib.WindowStepArgs(**{**step, **bad})), None) == code
    window = dict(dtype=0, comps=1, heads=2, kv_heads=1, head_channels=8, tile_rows=16, scale=1.0, n=4, num_graphs=1, longest=4, num_tiles=1, q=16, k=16, v=16, out=16, rest=16, tiles=16, ptr=16)
    for bad, code in ((dict(dtype=1), 1), (dict(tile_rows=8), 1), (dict(sinks=-1), 1), (dict(q=None), 1), (dict(n=2 ** 30), 2), (dict(head_channels=130), 2)):
        assert lib.eqt_window_attention_forward(C.byref(_lib.WindowAttentionArgs(**{**window, **bad})), None) == code
        assert bad.get("q", 1) is None or lib.eqt_window_attention_form(C.byref(_lib.WindowAttentionArgs(**{**window, **bad}))) == -1
    assert lib.eqt_window_attention_backward(C.byref(_lib.WindowAttentionArgs(**window)), None) == 1
    loss = dict(dtype=0, reduction=2, n=4, c=8, t=5, x=16, w=16, target=16, losses=16, lse=16, result=16, count=16, status=16)
    for bad, code in ((dict(dtype=1), 1), (dict(reduction=3), 1), (dict(c=0), 1), (dict(t=0), 1), (dict(x=None), 1), (dict(c=20_000), 2), (dict(scratch=16), 1)):
        assert lib.eqt_type_loss_forward(C.byref(_lib.TypeLossArgs(**{**loss, **bad})), None) == code
    assert lib.eqt_type_loss_backward(C.byref(_lib.TypeLossArgs(**loss)), None) == 1


def test_bfloat16_windows_keep_what_rounding_left():
    """Where the backward pass is to follow: its deltas go by it."""
    lib = _lib.lib()
    window = dict(dtype=_lib.DTYPE_CODE[torch.bfloat16], comps=1, heads=2, kv_heads=1, head_channels=8, tile_rows=16, scale=1.0, n=4, num_graphs=1, longest=4, num_tiles=1,
                  q=16, k=16, v=16, out=16, stats=16, tiles=16, ptr=16, grad=16, dq=16, dk=16, dv=16)
    assert lib.eqt_window_attention_forward(C.byref(_lib.WindowAttentionArgs(**window)), None) == 1
    assert lib.eqt_window_attention_backward(C.byref(_lib.WindowAttentionArgs(**window)), None) == 1
