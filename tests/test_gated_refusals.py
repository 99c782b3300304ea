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
    assert lib.eqt_gated_forward(9, 16, 16, 16, 1, 8, 8, 0, 16, None) == 1
    assert lib.eqt_gated_forward(0, 16, 16, 16, 1, 8, 8, 4, 16, None) == 1
    assert lib.eqt_gated_forward(0, 16, None, 16, 1, 8, 8, 0, 16, None) == 1
    assert lib.eqt_gated_forward(0, 16, 16, 16, 1, 8, 8, 0, None, None) == 1
    assert lib.eqt_gated_forward(0, 16, 16, 16, -1, 8, 8, 0, 16, None) == 1
    assert lib.eqt_gated_forward(0, 16, 16, 16, 2 ** 31, 8, 8, 0, 16, None) == 2
    assert lib.eqt_gated_forward(0, None, None, None, 0, 8, 8, 0, None, None) == 0
    assert lib.eqt_gated_backward(0, 16, 16, 16, 16, 16, None, 0, 4, 8, 8, 0, 16, None) == 1
