"""Which form of its kernel a gated layer runs, without a GPU (148 SMs are assumed where there is none)."""
from equitorch_b200 import _lib


def test_forms():
    form = _lib.lib().eqt_gated_form
    for sizes, forms in (((2, 100_000, 256, 1024), (2, 0, 1, 1)), ((2, 8192, 1024, 4096), (1, 1, 1, 1)), ((2, 40, 33_000, 8), (3, 3, 0, 1)),
                         ((2, 40, 8, 16_385), (0, 0, 3, 0)), ((0, 50_021, 64, 200), (2, 0, 0, 0)), ((0, 50_021, 65, 200), (0, 0, 0, 0)),
                         ((0, 40, 33_000, 8), (0, 0, 0, 0))):
        assert tuple(form(*sizes, product) for product in range(4)) == forms, sizes
    assert form(1, 10, 8, 8, 0) == -1 and form(2, 0, 8, 8, 0) == -1 and form(2, 10, 8, 8, 4) == -1 and form(2, 10, 8, 8, -1) == -1 and form(9, 10, 8, 8, 0) == -1
