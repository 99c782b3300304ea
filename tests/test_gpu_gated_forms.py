"""Every form of the gated layer's tensor-core kernel against the formulas in float64, at sizes that select it.

Forms, as ``eqt_gated_form`` names them, of the forward pass, the partial results, the gradient of x and that of the weights: 0 tiles of 128 rows,
1 pairs of CTAs, 2 weights held in shared memory, 3 sums in pieces."""
import pytest
import torch

from equitorch_b200 import _lib
from equitorch_b200.nn import functional as F

from .test_gpu_gated import _check, _inputs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16
CASES = [
    (BF16, 8200, 512, 1024, (1, 1, 1, 1)),           # eight rows in the last pair, its second CTA has none
    (BF16, 8192, 512, 512, (1, 1, 1, 1)),
    (BF16, 16129, 520, 301, (1, 1, 1, 1)),           # one row in the last pair, a last tile of 45 columns, rows that start anywhere
    (BF16, 8321, 515, 1030, (1, 1, 1, 1)),           # 129 rows in the last pair, both widths off 16 bytes
    (BF16, 5000, 1030, 2050, (1, 1, 1, 1)),
    (BF16, 4097, 640, 8192, (1, 1, 0, 1)),
    (BF16, 20000, 256, 512, (2, 0, 1, 1)),
    (BF16, 20000, 200, 300, (2, 0, 1, 1)),
    (BF16, 20011, 130, 515, (2, 0, 1, 1)),           # two channels in the second CTA's half of the weights' gradient
    (BF16, 20011, 300, 515, (0, 0, 1, 1)),
    (BF16, 3000, 136, 5000, (0, 0, 0, 1)),
    (BF16, 300, 33000, 70, (3, 3, 1, 1)),
    (BF16, 129, 40, 17001, (0, 0, 3, 0)),
    (F32, 50021, 64, 200, (2, 0, 0, 0)),
    (F32, 20011, 33, 130, (2, 0, 0, 0)),             # a second k-block of one channel, a last tile of two columns
    (F32, 30000, 40, 1000, (2, 0, 0, 0)),
    (F32, 40001, 64, 128, (2, 0, 0, 0)),
]


def _forms(dtype, rows, c, f):
    return tuple(_lib.lib().eqt_gated_form(_lib.DTYPE_CODE[dtype], rows, c, f, product) for product in range(4))


@pytest.mark.parametrize("dtype,rows,c,f,forms", CASES)
def test_forms(dtype, rows, c, f, forms):
    if torch.cuda.get_device_properties(0).multi_processor_count == 148:
        assert _forms(dtype, rows, c, f) == forms
    _check(*_inputs(rows, c, f, dtype), "silu")


@pytest.mark.parametrize("name", ["gelu", "relu", "sigmoid"])
@pytest.mark.parametrize("case", [3, 8, 14], ids=["pairs", "held", "held float32"])
def test_activations(case, name):
    dtype, rows, c, f, _ = CASES[case]
    _check(*_inputs(rows, c, f, dtype), name)


@pytest.mark.parametrize("case", [3, 7, 14], ids=["pairs", "held", "held float32"])
def test_rows_apart_and_same_bits_again(case):
    """A row that is not a number stays alone, and two calls give the same bits."""
    dtype, rows, c, f, _ = CASES[case]
    x, w, g = _inputs(rows, c, f, dtype)

    def run():
        h = F.gated_linear(x, w)
        return [h.detach(), *torch.autograd.grad(h, [x, w], g)]
    want, again = run(), run()
    assert all(torch.equal(a, b) for a, b in zip(want, again))
    with torch.no_grad():
        x[[130, rows - 1]] = float("nan")
    got = run()
    keep = torch.ones(rows, dtype=torch.bool, device=DEV)
    keep[[130, rows - 1]] = False
    assert all(torch.equal(a[keep], b[keep]) for a, b in zip(got[:2], want[:2])) and got[0][rows - 1].isnan().all()
