"""What the gated linear layer refuses, without a GPU."""
import pytest
import torch

from equitorch_b200 import _lib
from equitorch_b200 import nn as enn
from equitorch_b200.nn import functional as F


def test_refusals():
    x, w = torch.zeros(5, 8), torch.zeros(2, 8, 12)
    with pytest.raises(_lib.EqtError):
        F.gated_linear(x, w)
    for bad in ((x, w, "tanh"), (x, w[0]), (x, torch.zeros(3, 8, 12)), (torch.zeros(5, 7), w), (torch.zeros(()), w)):
        with pytest.raises(ValueError):
            F.gated_linear(*bad)
    for bad in ((x, w.double()), (x.half(), w.half()), (x.long(), w)):
        with pytest.raises(TypeError):
            F.gated_linear(*bad)
    with pytest.raises(ValueError):
        enn.GatedLinear(4, 8, "swish")


def test_library_checks_its_arguments():
    lib = _lib.lib()
    forward = lambda dtype=0, x=16, w=16, h=16, scratch=None, size=0, n=1, c=8, f=8, act=0, status=16: lib.eqt_gated_forward(  # noqa: E731
        dtype, x, w, h, scratch, size, n, c, f, act, status, None)
    assert forward(dtype=9) == 1 and forward(act=4) == 1 and forward(w=None) == 1 and forward(status=None) == 1 and forward(n=-1) == 1
    assert forward(n=2 ** 31) == 2 and forward(n=0, x=None, w=None, h=None, status=None) == 0
    assert forward(x=20) == 1 and b"16-byte" in lib.eqt_last_error()
    assert forward(c=7) == 1 and forward(c=7, scratch=16, size=8) == 1 and b"scratch" in lib.eqt_last_error()
    assert lib.eqt_gated_scratch(0, 1, 8, 8, 0) == 0 and lib.eqt_gated_scratch(0, 1, 7, 8, 0) > 0
    assert lib.eqt_gated_backward(0, 16, 16, 16, 16, 16, None, 0, 4, 8, 8, 0, 16, None) == 1
