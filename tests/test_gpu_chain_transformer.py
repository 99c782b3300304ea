"""Embedding, norms with the residual, rotary positions, attention within windows, gated products and the loss over types together, as a network over
packed chains trains and grows them."""
import threading

import pytest
import torch
from torch import nn

from equitorch_b200 import nn as enn
from equitorch_b200.graph import PackedGraphs
from equitorch_b200.nn import functional as F
from equitorch_b200.ops.fused_tp_op import check_status

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES, WIDTH, HEADS, KV, SIZE, HIDDEN = 37, 64, 4, 2, 16, 96
BEFORE, SINKS = 9, 2


class Block(nn.Module):
    def __init__(self):
        super().__init__()
        self.norm1, self.norm2 = enn.AddRMSNorm(WIDTH), enn.AddRMSNorm(WIDTH)
        self.qkv = nn.Parameter(torch.randn(WIDTH, (HEADS + 2 * KV) * SIZE) * WIDTH ** -0.5)
        self.out = nn.Parameter(torch.randn(HEADS * SIZE, WIDTH) * (HEADS * SIZE) ** -0.5)
        self.up = nn.Parameter(torch.randn(2, WIDTH, HIDDEN) * WIDTH ** -0.5)
        self.down = nn.Parameter(torch.randn(HIDDEN, WIDTH) * HIDDEN ** -0.5)
        self.attention = enn.WindowAttention(HEADS, BEFORE, 0, SINKS, KV)

    def project(self, x, stream, positions, frequencies):
        h, stream = self.norm1(x, stream)
        q, k, v = (h @ self.qkv).split([HEADS * SIZE, KV * SIZE, KV * SIZE], 2)          # views of one projection
        return (*F.rotary(q, k, positions, frequencies, HEADS, KV), v, stream)

    def finish(self, attended, stream):
        h, stream = self.norm2(attended @ self.out, stream)
        return F.gated_linear(h, self.up) @ self.down, stream

    def forward(self, x, stream, positions, frequencies, graphs):
        q, k, v, stream = self.project(x, stream, positions, frequencies)
        return self.finish(self.attention(q, k, v, graphs), stream)


class Network(nn.Module):
    def __init__(self, layers=2):
        super().__init__()
        self.embedding = enn.TypeEmbedding(TYPES, WIDTH)
        self.blocks = nn.ModuleList(Block() for _ in range(layers))
        self.norm, self.loss = enn.AddRMSNorm(WIDTH), enn.TypeCrossEntropy(TYPES, WIDTH)

    def features(self, types, positions, frequencies, graphs):
        x, stream = self.embedding(types), None
        for block in self.blocks:
            x, stream = block(x, stream, positions, frequencies, graphs)
        return self.norm(x, stream)[0][:, 0]

    def forward(self, types, target, positions, frequencies, graphs):
        return self.loss(self.features(types, positions, frequencies, graphs), target)


def plain(net, params, types, target, positions, frequencies, sizes):
    """The same in elementary operations, in the parameters' type."""
    p = dict(zip((n for n, _ in net.named_parameters()), params))
    dt = params[0].dtype

    def norm(h, w):
        return h / (h.square().mean(1, keepdim=True) + 1e-6).sqrt() * w

    def turn(x, heads):
        x = x.view(-1, heads, SIZE)
        angle = positions.double()[:, None] * frequencies
        cos, sin = torch.cos(angle).to(dt)[:, None], torch.sin(angle).to(dt)[:, None]
        a, b = x[..., :SIZE // 2], x[..., SIZE // 2:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], 2)

    graph = torch.repeat_interleave(torch.arange(len(sizes), device=DEV), torch.tensor(sizes, device=DEV))
    n = graph.numel()
    first = torch.tensor([0, *sizes], device=DEV).cumsum(0)[graph]
    i, j = torch.arange(n, device=DEV)[:, None], torch.arange(n, device=DEV)[None]
    mask = (graph[:, None] == graph[None]) & (j <= i) & ((j >= i - BEFORE) | (j < first[:, None] + SINKS))
    x, stream = p["embedding.weight"][types, 0], 0.0
    for b in range(len(net.blocks)):
        g = lambda name: p[f"blocks.{b}.{name}"]  # noqa: E731
        stream = x + stream
        q, k, v = (norm(stream, g("norm1.weight")) @ g("qkv")).split([HEADS * SIZE, KV * SIZE, KV * SIZE], 1)
        q, k, v = turn(q, HEADS), turn(k, KV).repeat_interleave(2, 1), v.reshape(n, KV, SIZE).repeat_interleave(2, 1)
        weight = (torch.einsum("ihc,jhc->hij", q, k) / SIZE ** 0.5).masked_fill(~mask, -torch.inf).softmax(2)
        stream = torch.einsum("hij,jhc->ihc", weight, v).reshape(n, -1) @ g("out") + stream
        h = norm(stream, g("norm2.weight"))
        a = h @ g("up")[0]
        x = (a * torch.sigmoid(a) * (h @ g("up")[1])) @ g("down")
    logits = norm(x + stream, p["norm.weight"]) @ p["loss.weight"].T
    counts = target >= 0
    return -(torch.log_softmax(logits, 1).gather(1, target.clamp(min=0)[:, None])[:, 0] * counts).sum() / counts.sum()


def make(sizes, seed=0):
    torch.manual_seed(seed)
    net = Network().to(DEV)
    n = sum(sizes)
    types = torch.randint(0, TYPES, (n,), device=DEV)
    target = torch.where(torch.rand(n, device=DEV) < 0.3, types, -1)
    positions = torch.cat([torch.arange(s) for s in sizes]).to(DEV)
    graphs = PackedGraphs(torch.tensor([0, *sizes], device=DEV).cumsum(0), n)
    return net, types, target, positions, F.rotary_frequencies(SIZE, device=DEV), graphs


def test_loss_and_gradients():
    """Against float64; as far from it as the same network of torch's float32 operations is, times eight: products of TF32 pairs lose 2^-21 of a term
    where float32 ones lose 2^-24."""
    sizes = (40, 1, 23, 90)
    net, types, target, positions, frequencies, graphs = make(sizes)
    loss = net(types, target, positions, frequencies, graphs)
    grads = torch.autograd.grad(loss, list(net.parameters()))
    results = {}
    for dt in (torch.float32, torch.float64):
        params = [p.detach().to(dt).requires_grad_(True) for p in net.parameters()]
        want = plain(net, params, types, target, positions, frequencies, sizes)
        results[dt] = [want.detach(), *torch.autograd.grad(want, params)]
    for got, single, exact in zip([loss.detach(), *grads], results[torch.float32], results[torch.float64]):
        exact = exact.view(got.shape)
        size = exact.norm().item()
        assert (got.double() - exact).norm().item() <= 8 * (single.view(got.shape).double() - exact).norm().item() + 2.0 ** -22 * size
    check_status()


def test_growing_chains_by_a_node_at_a_time():
    """The features of a chain that grows over a cache are those of the whole chain, node by node."""
    length = 30
    net, types, _, positions, frequencies, graphs = make((length, length))
    with torch.no_grad():
        want = net.features(types, positions, frequencies, graphs).view(2, length, WIDTH)
        caches = [torch.zeros(2, 2, length + 3, 1, KV * SIZE, device=DEV) for _ in net.blocks]
        for at in range(length):
            x, stream = net.embedding(types.view(2, length)[:, at]), None
            place, lengths = torch.full((2,), at, device=DEV), torch.full((2,), at + 1, device=DEV)
            for block, (keys, values) in zip(net.blocks, caches):
                q, keys[:, at], values[:, at], stream = block.project(x, stream, place, frequencies)
                x, stream = block.finish(F.window_attention_step(q, keys, values, lengths, HEADS, BEFORE, SINKS, KV), stream)
            got = net.norm(x, stream)[0][:, 0]
            assert (got - want[:, at]).norm() <= 1e-5 * want[:, at].norm()          # float32's error of a layer, a few times


def test_training_step_in_a_cuda_graph():
    net, types, target, positions, frequencies, graphs = make((40, 7))
    params = list(net.parameters())
    step = lambda: torch.autograd.grad(net(types, target, positions, frequencies, graphs), params)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    target.copy_(torch.where(target < 0, types, target))
    graph.replay()
    again = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, again))


def test_bfloat16_trains():
    net, types, target, positions, frequencies, graphs = make((40, 1, 23, 90))
    wide = torch.autograd.grad(net(types, target, positions, frequencies, graphs), list(net.parameters()))
    net = net.bfloat16()
    narrow = torch.autograd.grad(net(types, target, positions, frequencies, graphs), list(net.parameters()))
    for a, b in zip(narrow, wide):                           # some twenty roundings of 2^-8 between the types and the loss
        assert torch.isfinite(a).all() and (a.float() - b).norm() <= 20 * 2.0 ** -8 * b.norm()


def test_threads_on_streams_of_their_own():
    """Each operator from several host threads at once, each on a stream of its own: the same bits."""
    gen = torch.Generator(device=DEV).manual_seed(0)
    rand = lambda *s, dtype=torch.bfloat16: torch.randn(*s, device=DEV, generator=gen).to(dtype)  # noqa: E731
    graphs = PackedGraphs(torch.tensor([0, 300, 301, 900], device=DEV), 900)

    def attention(dtype, size):
        q, k, v, g = rand(900, 1, 4 * size, dtype=dtype), rand(900, 1, 2 * size, dtype=dtype), rand(900, 1, 2 * size, dtype=dtype), rand(900, 1, 4 * size, dtype=dtype)
        leaves = [t.requires_grad_(True) for t in (q, k, v)]

        def call():
            out = F.window_attention(*leaves, graphs, 4, 50, 3, 2, kv_heads=2)
            return [out.detach(), *torch.autograd.grad(out, leaves, g)]
        return call

    def loss(dtype):
        x, w, target = rand(500, 72, dtype=dtype).requires_grad_(True), rand(3000, 72, dtype=dtype).requires_grad_(True), torch.randint(0, 3000, (500,), device=DEV)

        def call():
            out = F.type_cross_entropy(x, w, target)
            return [out.detach(), *torch.autograd.grad(out, [x, w])]
        return call

    def norm():
        x, w, g = rand(2000, 3, 64).requires_grad_(True), rand(64).requires_grad_(True), rand(2000, 3, 64)

        def call():
            out, total = F.add_rms_norm(x, x.detach(), w)
            return [out.detach(), total.detach(), *torch.autograd.grad(out, [x, w], g), *(t.float() for t in F.add_rms_norm_e4m3(x.detach(), None, w.detach(), group=32)[:2])]
        return call

    def step():
        q, keys, values, lengths = rand(20, 1, 128), rand(20, 400, 1, 64), rand(20, 400, 1, 64), torch.randint(1, 400, (20,), device=DEV)
        frequencies = F.rotary_frequencies(32, device=DEV)
        return lambda: [F.window_attention_step(q, keys, values, lengths, 4, 200, 2, kv_heads=2), F.rotary(q, None, lengths, frequencies, 4)]

    calls = [attention(torch.bfloat16, 64), attention(torch.float32, 32), attention(torch.bfloat16, 128), loss(torch.bfloat16), loss(torch.float32), norm(), step()]
    want, errors = [call() for call in calls], []
    torch.cuda.synchronize()

    def work(call, ref):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(30):
                    assert all(torch.equal(a, b) for a, b in zip(call(), ref))
        except Exception as e:                                   # noqa: BLE001 - handed to the main thread
            errors.append(e)
    threads = [threading.Thread(target=work, args=pair) for pair in zip(calls, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    check_status()
