"""Weights of bfloat16 windows are rounded alike in the forward pass and by rows, whatever the unit of the moment was."""
import math

import pytest
import torch

from equitorch_b200.graph import PackedGraphs
from equitorch_b200.nn import functional as F
from equitorch_b200.ops.fused_tp_op import check_status

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("sign", [1.0, -1.0])               # tiles of 128 nodes, and of one chain
@pytest.mark.parametrize("size", [16, 64, 128])
@pytest.mark.parametrize("rise", [(0.0, 7.75, 8.1875), (0.0, 7.75, 8.1875, 16.75), (0.3125, 0.8125, 1.4375, 2.1875, 9.0625), (-3.0, 4.5, 5.375, 5.75, 0.0)])
def test_score_gradients_of_a_row_cancel(rise, size, sign):
    """Scores rise along the chain, 64 nodes at a time, so that earlier weights were rounded in another unit than the last one.  A row's score gradients add up to zero if its
    weights and those in its delta are the same, else to 4e-4 where one is rounded in two ways.  Deltas go by the result and what its rounding left, 2^-17 of it; score
    gradients go into the product in two parts, 2^-17 of them, whose absolute values add up to one at most; sums lose 2^-19."""
    n = 64 * len(rise)
    q, k, v = (torch.zeros(n, 1, size, device=DEV, dtype=torch.bfloat16) for _ in range(3))
    q[:, :, 0] = sign
    k[:, 0, 0] = torch.tensor(rise, device=DEV).bfloat16().repeat_interleave(64)
    k[:, :, 1] = 1.0                                        # whose product with the score gradients is their sum
    v[:, 0, 0] = 1.0 - 2.0 * (torch.arange(n, device=DEV) // 64 % 2)
    g = torch.zeros_like(v)
    g[:, :, 0] = 1.0
    graphs = PackedGraphs(torch.tensor([0, n], device=DEV), n)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = F.window_attention(*leaves, graphs, 1, n, n, scale=sign * math.log(2))
    (dq,) = torch.autograd.grad(out, q, g)
    assert dq[:, :, 1].abs().max() <= math.log(2) * 2.0 ** -15
    check_status()


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("size", [16, 64, 128])
def test_scores_far_apart(size, sign):
    """From -2e6 to 2e6 in units of log2: the row goes by the greatest, and by those before where these are all there is."""
    n, high = 192, 1024.0
    q, k, v = (torch.zeros(n, 1, size, device=DEV, dtype=torch.bfloat16) for _ in range(3))
    q[:, :, 0] = sign * high
    k[:, 0, 0] = torch.tensor([-high, high, -high], device=DEV).repeat_interleave(64)
    v[:, 0, 0] = torch.tensor([1.0, 2.0, 4.0], device=DEV).repeat_interleave(64)
    graphs = PackedGraphs(torch.tensor([0, n], device=DEV), n)
    out = F.window_attention(q, k, v, graphs, 1, n, 0, scale=sign * 1.4)
    assert (out[:64, 0, 0] == 1).all() and (out[64:, 0, 0] == 2).all()
    check_status()
