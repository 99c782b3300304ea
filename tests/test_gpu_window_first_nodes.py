"""First nodes of chains some of which are long enough that queries behind a window are taken apart, and others not, next to each other in a batch."""
import pytest
import torch

from equitorch_b200.ops.fused_tp_op import check_status

from .test_gpu_window import compare, make, run
from .window_reference import reference, seen

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def no_wait_gave_up():
    yield
    check_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("before,after,sinks", [(30, 2, 4), (0, 0, 1), (100, 0, 40)])
@pytest.mark.parametrize("size", [16, 64])
def test_chains_about_the_length_from_which_they_are_taken_apart(size, before, after, sinks, dtype):
    edge = before + 1 + 512
    sizes = (edge - 1, edge, 0, 5, edge + 1, 511, 1, edge + 1300, 2, edge, edge, edge - 1)
    n = sum(sizes)
    qkv, g, graphs = make(sizes, 1, 4, 2, size, dtype, seed=before)
    want, bound = reference(*qkv, g, seen(sizes, n, before, after, sinks), 4, 2, None)
    compare(run(qkv, g, graphs, 4, before, after, sinks, kv_heads=2), want, bound)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_long_chain_among_many_short_ones(dtype):
    """Its gradients are those that it has alone; scratch is in proportion to the nodes."""
    sizes = (10,) * 7000 + (3000,) + (17,) * 13_000
    qkv, g, graphs = make(sizes, 1, 4, 4, 32, dtype)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    start = torch.cuda.memory_allocated()
    got = run(qkv, g, graphs, 4, 30, 0, 4)
    peak = torch.cuda.max_memory_allocated() - start
    # results, what rounding left and three gradients; statistics, deltas and their like, the nodes' chains; what queries far behind give first nodes: 0.55 of a byte a value
    n, row = sum(sizes), 4 * 32
    assert peak <= n * (5 * row * qkv[0].element_size() + 4 * 4 * 4 + 8 + 0.55 * row) + 8 * 2 ** 20
    lo, hi = 70_000, 73_000
    part = [t.detach()[lo:hi].clone().requires_grad_(True) for t in qkv]
    want, bound = reference(*part, g[lo:hi], seen((3000,), 3000, 30, 0, 4), 4, 4, None)
    compare([t[lo:hi] for t in got], want, bound)
