"""How far bfloat16 gradients of attention are off in the mean, and that they do not go by who else wants one."""
import math

import pytest
import torch

from equitorch_b200.nn import functional as F

from .test_gpu_attention import _inputs, _reference, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sizes", [[150] * 20, [700], [40, 250, 90, 16]])
@pytest.mark.parametrize("bias,cap", [(False, None), (False, 20.0), (True, 20.0)])
def test_error_in_the_mean(sizes, bias, cap):
    """dq has the rounding of the result; out, dk and dv have that of the weights or score gradients too.  dq also goes by delta = <g, out> of rounded
    weights and outputs: delta is off by their two roundings times the norm of the outputs, next to which the gradient of the scores, <g, v> - delta,
    has the norm of the values; scores are flat here (a scale of 0.3 over the root of the values), so outputs are a third of the values at most.
    What one rounding is in the mean is taken from the definition; 5 % are for sizes of few values."""
    leaves, cot, graphs = _inputs(sizes, 1, 4, 64, torch.bfloat16, bias, spread=0.5)
    got = _run(leaves, cot, graphs, 4, 0.3 / 8, cap)
    want, _ = _reference(leaves, cot, graphs, 4, 0.3 / 8, cap)
    for name, x, y, roundings in zip(("out", "dq", "dk", "dv"), got, want, (2, 1 + 2 / 9, 2, 2)):
        error, one = (float((z.double() - y).norm() / y.norm()) for z in (x, y.bfloat16()))
        assert error <= 1.05 * math.sqrt(roundings) * one, f"{name}: {error:.3g}, one rounding {one:.3g}"


@pytest.mark.parametrize("sizes", [[30, 60, 7], [300, 500]])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_of_features_with_and_without_those_of_positions(dtype, sizes):
    leaves, cot, graphs = _inputs(sizes, 1, 2, 32, dtype, True)
    q, k, v, pos, slope = leaves
    all_of_them = _run(leaves, cot, graphs, 2, 0.2, 10.0)
    out = F.graph_attention(q, k, v, graphs, 2, 0.2, 10.0, pos.detach(), slope.detach())
    few = torch.autograd.grad(out, [q, k, v], cot)
    assert all(torch.equal(a, b) for a, b in zip(few, all_of_them[1:4]))
