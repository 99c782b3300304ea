"""Attention within graphs, gated products and type embeddings from several host threads at once, each on a stream of its own."""
import threading

import pytest
import torch

from equitorch_b200.graph import PackedGraphs
from equitorch_b200.nn import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _attention(size):
    n = 40 * size
    q, k, v = (torch.randn(n, 1, 2 * size, device=DEV, dtype=torch.bfloat16, requires_grad=True) for _ in range(3))
    pos, slope = torch.rand(n, 3, device=DEV, requires_grad=True), torch.rand(2, device=DEV, requires_grad=True)
    cot, ptr = torch.randn(n, 1, 2 * size, device=DEV, dtype=torch.bfloat16), torch.tensor([0, 7, n // 2, n], device=DEV)

    def call():
        out = F.graph_attention(q, k, v, PackedGraphs(ptr, n), 2, 0.1, 30.0, pos, slope)
        return [out.detach(), *torch.autograd.grad(out, [q, k, v, pos, slope], cot)]
    return call


def _gated(rows, c, f, dtype):
    x, w = torch.randn(rows, c, device=DEV, dtype=dtype, requires_grad=True), torch.randn(2, c, f, device=DEV, dtype=dtype, requires_grad=True)
    cot = torch.randn(rows, f, device=DEV, dtype=dtype)

    def call():
        h = F.gated_linear(x, w)
        return [h.detach(), *torch.autograd.grad(h, [x, w], cot)]
    return call


def _embedding(rows):
    index, w = torch.randint(0, 200, (rows,), device=DEV), torch.randn(200, 48, device=DEV, requires_grad=True)
    cot = torch.randn(rows, 48, device=DEV)

    def call():
        out = F.type_embedding(index, w, 0.5)
        return [out.detach(), *torch.autograd.grad(out, [w], cot)]
    return call


def test_threads_on_streams_of_their_own():
    torch.manual_seed(0)
    calls = [_attention(32), _attention(64), _gated(5000, 64, 200, torch.float32), _gated(20000, 256, 512, torch.bfloat16), _gated(700, 33, 70, torch.bfloat16),
             _embedding(30000)]
    want, errors = [call() for call in calls], []
    torch.cuda.synchronize()

    def work(call, ref):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(40):
                    got = call()
                    assert all(torch.equal(a, b) for a, b in zip(got, ref))
        except Exception as e:                                   # noqa: BLE001 - handed to the main thread
            errors.append(e)
    threads = [threading.Thread(target=work, args=pair) for pair in zip(calls, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
