"""Values that are not finite, and rows that do not see them: others on the far side keep their bits, near ones are within their bounds."""
import pytest
import torch

from equitorch_b200.ops.fused_tp_op import check_status

from .test_gpu_window import make, run
from .window_reference import reference, seen

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("which", [0, 1, 2, 3])
def test_rows_that_do_not_see_it(which, value, dtype):
    sizes, (before, after, sinks), at = (1000, 90), (20, 3, 2), 500
    n = sum(sizes)
    qkv, g, graphs = make(sizes, 1, 2, 1, 64, dtype)
    mask = seen(sizes, n, before, after, sinks).to(DEV)
    clean = run(qkv, g, graphs, 2, before, after, sinks, kv_heads=1)
    want, bound = reference(*qkv, g, mask, 2, 1, None)
    bad = [t.detach().clone() for t in (*qkv, g)]
    bad[which][at, 0, 5] = value
    got = run([t.requires_grad_(True) for t in bad[:3]], bad[3], graphs, 2, before, after, sinks, kv_heads=1)
    rows = torch.zeros(n, dtype=torch.bool, device=DEV)
    rows[at] = True
    hit = rows if which in (0, 3) else mask[:, at]          # rows whose result the value is in
    keys = mask[hit].any(0)                                 # and the keys whose gradients these are in, first nodes among them
    place = torch.arange(n, device=DEV)
    far = (place - at).abs() > 128 + 64 + before            # no tile of 128 nodes, and no step of 64 that it takes, has the value and such a row
    first = place < 128                                     # by columns, the tile (of 64 nodes, or of 128) with a chain's first nodes meets all of the chain
    for a, b, w, e, h, near in zip(got, clean, want, bound, (hit if which != 3 else rows & False, hit, keys, keys), (~far, ~far, ~far | first, ~far | first)):
        assert torch.equal(a[~near & ~h], b[~near & ~h])
        assert ((a.double() - w).abs() - e)[~h].max() <= 1e-30
    check_status()


@pytest.mark.parametrize("size", [32, 64, 128])
@pytest.mark.parametrize("window", [(2, 1, 1), (30, 30, 4), (200, 0, 0)])
def test_gradients_of_keys_and_values_of_few_tiles(window, size):
    """bfloat16: no more tiles than SMs, so weights and score gradients go in two parts, which leave 2^-17, and a result's rounding, 1.66e-3 of its 2-norm, is all; a tenth for
    what some hundred rows vary."""
    sizes = (150, 3, 90, 257)
    qkv, g, graphs = make(sizes, 1, 4, 2, size, torch.bfloat16, seed=size)
    want, _ = reference(*qkv, g, seen(sizes, sum(sizes), *window), 4, 2, None)
    for what, a, b in zip(("dk", "dv"), run(qkv, g, graphs, 4, *window, kv_heads=2)[2:], want[2:]):
        error = ((a.double() - b).norm() / b.norm()).item()
        assert error < 1.1 * 1.66e-3, f"{what}: {error:.2e}"
