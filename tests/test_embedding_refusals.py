"""What the type embedding refuses, without a GPU."""
import pytest
import torch

from equitorch_b200 import _lib
from equitorch_b200.nn import functional as F


def test_refusals():
    index, table = torch.zeros(3, dtype=torch.int64), torch.zeros(5, 4)
    with pytest.raises(_lib.EqtError):
        F.type_embedding(index, table)
    with pytest.raises(TypeError, match="int64"):
        F.type_embedding(index.int(), table)
    with pytest.raises(TypeError, match="float32"):
        F.type_embedding(index, table.half())
    with pytest.raises(ValueError, match="types"):
        F.type_embedding(index, table[:, 0])


def test_library_checks_its_arguments():
    lib = _lib.lib()
    assert lib.eqt_embedding_forward(7, 16, 16, 16, 1, 1, 4, 1.0, None) == 1
    assert lib.eqt_embedding_forward(0, 16, 16, 16, -1, 1, 4, 1.0, None) == 1
    assert lib.eqt_embedding_forward(0, 16, None, 16, 1, 1, 4, 1.0, None) == 1
    assert lib.eqt_embedding_forward(0, 16, 16, 16, 2 ** 31, 1, 4, 1.0, None) == 2
    assert lib.eqt_embedding_forward(0, 16, 16, 16, 1, 1, 2 ** 20 + 1, 1.0, None) == 2
    assert lib.eqt_embedding_grad(0, None, 16, 16, 1, 1, 4, 1.0, None, 0, None) == 1
    assert lib.eqt_embedding_grad(0, 16, 16, 16, 1, 2 ** 31, 4, 1.0, None, 0, None) == 2
