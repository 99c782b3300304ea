"""What the norms refuse besides, without a GPU."""
import pytest
import torch

from equitorch_b200 import _lib
from equitorch_b200.nn import functional as F


@pytest.mark.parametrize("eps", [1e-50, 5e-324, 1e39, 1e300])
def test_eps_that_float32_does_not_have(eps):
    """It would be zero, and a row of zeros NaN, or infinite, and all results zero."""
    x, w = torch.zeros(4, 2, 8), torch.ones(8)
    for call in (F.add_rms_norm, F.add_rms_norm_e4m3):
        with pytest.raises(ValueError, match="eps"):
            call(x, None, w, eps)
    lib = _lib.lib()
    assert lib.eqt_add_rms_norm_forward(0, 16, None, 16, 16, None, None, 1, 1, 8, eps, None) == 1
    assert lib.eqt_add_rms_norm_e4m3(0, 16, None, 16, 16, 16, None, 1, 1, 8, 8, eps, None) == 1
