"""Scratch of the cross entropy's backward pass, without a GPU: logits' gradients of a piece of the types, one float32 gradient of the features, and operands."""
import ctypes as C

import pytest
import torch

from equitorch_b200 import _lib

MB = 2 ** 20


def scratch(n, t, c, dtype=torch.bfloat16, dx=16, dw=16):
    args = _lib.TypeLossArgs(dtype=_lib.DTYPE_CODE[dtype], reduction=2, n=n, c=c, t=t, x=16, w=16, target=16, lse=16, count=16, status=16, grad=16, dx=dx, dw=dw)
    return _lib.lib().eqt_type_loss_scratch(C.byref(args), 1)


@pytest.mark.parametrize("n", [16_384, 65_536, 131_072])
@pytest.mark.parametrize("c", [512, 4096])
def test_it_does_not_grow_with_the_table(n, c):
    sizes = [scratch(n, t, c) for t in (32_768, 131_072, 1_000_000)]
    # The features' copy and their gradient; of a piece's p types, whose logits' gradients are 2 n p <= 256 MB, the table's gradient in parts of 16,384 rows: n / 16,384
    # times 4 p c, at most 32,768 c; or in more parts where tiles are few.
    assert max(sizes) <= 256 * MB + n * c * 2 + n * c * 4 + 32_768 * c + 64 * MB


def test_float32_has_operands_in_three_parts_besides():
    n, t, c = 131_072, 32_768, 512
    assert scratch(n, t, c, torch.float32) <= 256 * MB + (n + t) * c * 6 + n * c * 4 + 32_768 * c + 64 * MB


def test_what_is_not_wanted_takes_none():
    n, t, c = 65_536, 131_072, 1024
    assert scratch(n, t, c) - scratch(n, t, c, dx=None) >= n * c * 4
    n, t, c = 40_000, 100, 64                               # few tiles: the table's gradient in parts
    assert scratch(n, t, c, dw=None) < scratch(n, t, c)
