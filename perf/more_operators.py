"""The operators of a pre-norm transformer over packed chains (residues, monomers, atoms in their order), and what they are timed on: the
calls that a user makes, their plain forms in elementary torch operations, and their definitions in 64 bits.

norm      ``add_rms_norm``: the residual's addition and the root-mean-square norm of a node's values over all components and channels;
          ``add_rms_norm_e4m3``: the same with the result in 8 bits and scales
rotary    ``rotary``: channel pairs of every head of q and k turned by angles that go with the node's position along its chain
window    ``window_attention``: a node attends to the nodes up to ``before`` behind and ``after`` ahead of it in its own chain, and to the
          chain's first ``sinks`` ones; heads may share keys and values
step      ``window_attention_step``: the same for one new node of every chain, over a cache
loss      ``type_cross_entropy``: cross entropy over the types of a table, without keeping the logits
"""
from __future__ import annotations

import math
import random
from types import SimpleNamespace

import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-6
E4M3_MAX = 448.0


def listed():
    return [
        # A small training batch, 32 molecules of 30 atoms: launches and latency count.
        dict(name="norm_f32_960", kind="norm", type="f32", rows=960, comps=1, channels=128, residual=True, group=-1, train=True),
        # The stream of a large training step of equivariant features 0e+1o: four components, ragged count of nodes.
        dict(name="norm_bf16_equivariant_100k", kind="norm", type="bf16", rows=100_003, comps=4, channels=256, residual=True, group=-1,
             train=True),
        # In front of an 8-bit product at inference: a scale for every 128 channels.
        dict(name="norm_e4m3_32k", kind="norm", type="bf16", rows=32_768, comps=1, channels=2048, residual=True, group=128, train=False),
        # Queries and keys of a large training step over chains, eight heads sharing two heads of keys.
        dict(name="rotary_bf16_65k", kind="rotary", type="bf16", rows=65_536, comps=1, heads=8, kv_heads=2, size=64, rotated=64,
             interleaved=False, far=2_000, train=True),
        # One new node of 32 chains, half of each head turned, pairs next to each other, positions far out.
        dict(name="rotary_f32_32", kind="rotary", type="f32", rows=32, comps=1, heads=4, kv_heads=4, size=32, rotated=16,
             interleaved=True, far=1_000_000, train=False),
        # Chains of 30 nodes with equivariant features 0e+1o, float32.
        dict(name="window_f32_32x30", kind="window", type="f32", graphs=32, low=30, high=30, comps=4, heads=4, kv_heads=4, size=16,
             before=8, after=8, sinks=1, train=True),
        # Proteins of 50 to 500 residues seen from both sides, four heads of queries to one of keys.
        dict(name="window_bf16_proteins", kind="window", type="bf16", graphs=240, low=50, high=500, comps=1, heads=8, kv_heads=2, size=64,
             before=64, after=64, sinks=4, train=True),
        # One long chain read in its order.
        dict(name="window_bf16_long_chain", kind="window", type="bf16", graphs=1, low=32_781, high=32_781, comps=1, heads=8, kv_heads=8,
             size=128, before=1023, after=0, sinks=4, train=True),
        # Growing 64 chains by a node each, from a cache of 8192 nodes a chain.
        dict(name="step_bf16_64", kind="step", type="bf16", graphs=64, capacity=8192, high=8192, comps=1, heads=16, kv_heads=4, size=64,
             before=4095, sinks=4, train=False),
        # Masked atom types of the small batch.
        dict(name="loss_f32_960", kind="loss", type="f32", rows=960, types=119, channels=128, ignored=0.1, train=True),
        # Pairs of atom types: many types, ragged sizes, float32.
        dict(name="loss_f32_pairs", kind="loss", type="f32", rows=5_003, types=14_161, channels=128, ignored=0.1, train=True),
        # Structure tokens of a large training step.
        dict(name="loss_bf16_tokens", kind="loss", type="bf16", rows=16_384, types=32_768, channels=512, ignored=0.0, train=True),
    ]


def _log(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return min(hi, n | 1) if rng.random() < 0.5 else n


def draw(rng):
    kind = rng.choice(["norm", "norm", "rotary", "rotary", "window", "window", "window", "step", "loss", "loss", "loss"])
    type_ = rng.choice(["f32", "bf16"])
    train = rng.random() < 0.75
    if kind == "norm":
        comps = rng.choice([1, 1, 1, 4, 9])
        channels = rng.choice([rng.randint(8, 300), 64, 128, 256, 512, 16 * rng.randint(1, 150)])
        group = -1 if train or rng.random() < 0.4 else rng.choice([0, 0, 128])
        if group == 128:
            comps, channels = 1, 128 * rng.randint(1, 24)
        rows = max(1, min(_log(rng, 1, 200_000), int(4.0e7 / (comps * channels))))
        return dict(kind=kind, type=type_, rows=rows, comps=comps, channels=channels, residual=rng.random() < 0.7, group=group,
                    train=train)
    if kind == "rotary":
        comps, size = rng.choice([1, 1, 4]), rng.choice([8, 16, 32, 64, 64, 128, 20, 6])
        heads = rng.choice([1, 2, 4, 8, 12])
        kv_heads = rng.choice([h for h in (1, 2, 3, 4, 8, 12) if heads % h == 0])
        rows = max(1, min(_log(rng, 1, 100_000), int(2.5e7 / (comps * (heads + kv_heads) * size))))
        return dict(kind=kind, type=type_, rows=rows, comps=comps, heads=heads, kv_heads=kv_heads, size=size,
                    rotated=size if rng.random() < 0.6 else 2 * rng.randint(1, size // 2), interleaved=rng.random() < 0.5,
                    far=rng.choice([100, 10_000, 2_000_000]), train=train)
    if kind == "step":
        comps, size = rng.choice([(1, 16), (1, 32), (1, 64), (1, 64), (1, 128), (4, 16)])
        kv_heads = rng.choice([1, 2, 4])
        heads = kv_heads * rng.choice([1, 1, 2, 4, 6])
        high = _log(rng, 1, 16_000)
        graphs = max(1, min(_log(rng, 1, 128), int(1.2e8 / (high * comps * kv_heads * size))))
        return dict(kind=kind, type=type_, graphs=graphs, capacity=high + rng.choice([0, 1, 100]), high=high, comps=comps, heads=heads,
                    kv_heads=kv_heads, size=size, before=rng.choice([0, 100, 511, 4095, 16_000]), sinks=rng.choice([0, 1, 4]),
                    train=False)
    if kind == "window":
        comps, size = rng.choice([(1, 8), (1, 16), (1, 32), (1, 64), (1, 64), (1, 128), (4, 8), (4, 16), (9, 8)])
        kv_heads = rng.choice([1, 2, 4])
        heads = kv_heads * rng.choice([1, 1, 2, 4])
        before = rng.choice([3, 16, 64, 127, 256, 500, 1023])   # a node that sees itself alone has no gradient of q and k
        after = rng.choice([0, 0, before, 1, 17])
        high = _log(rng, 8, 8_000)
        low = rng.choice([0, 1, high // 8, high // 2, high])
        band = min(high, before + after + 128)
        most = 1.2e10 / (band * heads * comps * size) / (8 if type_ == "f32" else 1)
        graphs = max(1, min(_log(rng, 1, 1000), int(most / high), int(2.0e7 / (high * comps * heads * size))))
        high = max(1, min(high, int(most)))
        return dict(kind=kind, type=type_, graphs=graphs, low=min(low, high), high=high, comps=comps, heads=heads, kv_heads=kv_heads,
                    size=size, before=before, after=after, sinks=rng.choice([0, 1, 4]), train=train)
    channels = rng.choice([rng.randint(8, 200), 64, 128, 256, 512, _log(rng, 32, 1024)])
    types = _log(rng, 2, 33_000)
    most = 1.1e11 / (channels * types) / (4 if type_ == "f32" else 1)
    return dict(kind=kind, type=type_, rows=max(1, min(_log(rng, 1, 20_000), int(most))), types=types, channels=channels,
                ignored=rng.choice([0.0, 0.0, 0.15]), train=train)


def _sizes(case):
    """Nodes of each chain, ascending counts shuffled by the case's own numbers (not by the seed: `work` counts them too)."""
    low, high, graphs = case["low"], case["high"], case["graphs"]
    sizes = [low + (high - low) * i // max(1, graphs - 1) for i in range(graphs)] if graphs > 1 else [high]
    random.Random(graphs * 7919 + high).shuffle(sizes)
    return sizes


def _lengths(case):
    """Nodes of each chain in the cache, the new one among them."""
    rng = random.Random(case["graphs"] * 104_729 + case["high"])
    return [case["high"]] + [rng.randint(1, case["high"]) for _ in range(case["graphs"] - 1)]


def _seen(n, before, after, sinks):
    """Pairs of nodes that see each other in a chain of n nodes."""
    i = torch.arange(n)
    low, high = (i - before).clamp(min=0), (i + after).clamp(max=n - 1)
    return int((high - low + 1 + torch.minimum(low, torch.full_like(low, sinks))).sum())


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = TYPES[case["type"]]
    rand = lambda *shape: torch.randn(*shape, device=DEV, generator=g)  # noqa: E731
    s = SimpleNamespace(case=case)
    kind, train = case["kind"], case["train"]
    if kind == "norm":
        shape = (case["rows"], case["comps"], case["channels"])
        s.x = rand(*shape).to(dt)
        # the stream has grown over the layers before, channels differ in scale
        s.residual = (3.0 * rand(*shape) * (0.5 + torch.rand(case["channels"], device=DEV, generator=g))).to(dt) if case["residual"] else None
        s.weight = (1.0 + 0.2 * rand(case["channels"])).to(dt)
        s.cots = [rand(*shape).to(dt) for _ in range(2)] if train else None
        s.leaves = [t for t in (s.x, s.residual, s.weight) if t is not None]
    elif kind == "rotary":
        shape = lambda heads: (case["rows"], case["comps"], heads * case["size"])  # noqa: E731
        s.q, s.k = rand(*shape(case["heads"])).to(dt), rand(*shape(case["kv_heads"])).to(dt)
        s.positions = torch.randint(0, case["far"], (case["rows"],), device=DEV, generator=g)
        half = case["rotated"] // 2
        s.frequencies = 10_000.0 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)
        s.cots = [rand(*t.shape).to(dt) for t in (s.q, s.k)] if train else None
        s.leaves = [s.q, s.k]
    elif kind == "window":
        sizes = _sizes(case)
        n, d = sum(sizes), case["comps"]
        s.ptr = torch.tensor([0] + sizes, device=DEV).cumsum(0)
        s.q = (1.5 * rand(n, d, case["heads"] * case["size"])).to(dt)
        s.k, s.v = (rand(n, d, case["kv_heads"] * case["size"]).to(dt) for _ in range(2))
        s.cots = [rand(*s.q.shape).to(dt)] if train else None
        if own:
            from equitorch_b200.graph import PackedGraphs
            s.graphs = PackedGraphs(s.ptr, n)
        s.leaves = [s.q, s.k, s.v]
    elif kind == "step":
        d, cache = case["comps"], (case["graphs"], case["capacity"], case["comps"], case["kv_heads"] * case["size"])
        s.q = (1.5 * rand(case["graphs"], d, case["heads"] * case["size"])).to(dt)
        s.k, s.v = rand(*cache).to(dt), rand(*cache).to(dt)
        s.lengths = torch.tensor(_lengths(case), device=DEV)
        s.leaves = []
    else:
        c, t = case["channels"], case["types"]
        s.x, s.weight = rand(case["rows"], c).to(dt), (1.5 * rand(t, c) / math.sqrt(c)).to(dt)
        # type frequencies fall off with their rank, the types in no order; nodes that do not count have no type
        prob = torch.arange(1, t + 1, device=DEV, dtype=torch.float64).pow(-0.8)
        rank = torch.searchsorted((prob.cumsum(0) / prob.sum()).float(), torch.rand(case["rows"], device=DEV, generator=g)).clamp_(max=t - 1)
        s.target = torch.randperm(t, device=DEV, generator=g)[rank]
        s.target[torch.rand(case["rows"], device=DEV, generator=g) < case["ignored"]] = -1
        s.cots = None
        s.leaves = [s.x, s.weight]
    if train:
        for leaf in s.leaves:
            leaf.requires_grad_(True)
    return s


def run(s):
    if own:
        outs = _call(s)
        if not s.case["train"]:
            return outs
        return [*outs, *torch.autograd.grad(outs, s.leaves, s.cots)]
    dt, train = TYPES[s.case["type"]], s.case["train"]
    if not train:
        return _plain(s, s.leaves)
    wide = [t.detach().float().requires_grad_(True) for t in s.leaves]
    outs = _plain(s, wide)
    grads = torch.autograd.grad(outs, wide, None if s.cots is None else [c.float() for c in s.cots])
    return [*(o.detach() if s.case["kind"] == "loss" else o.detach().to(dt) for o in outs), *(a.to(b.dtype) for a, b in zip(grads, s.leaves))]


def _call(s):
    from equitorch_b200.nn import functional as F
    case = s.case
    if case["kind"] == "norm":
        if case["group"] < 0:
            return list(F.add_rms_norm(s.x, s.residual, s.weight, EPS))
        values, scales, total = F.add_rms_norm_e4m3(s.x, s.residual, s.weight, EPS, group=case["group"] or None)
        return [_spread(values.float(), scales), total]
    if case["kind"] == "rotary":
        return list(F.rotary(s.q, s.k, s.positions, s.frequencies, case["heads"], case["kv_heads"], interleaved=case["interleaved"]))
    if case["kind"] == "window":
        return [F.window_attention(s.q, s.k, s.v, s.graphs, case["heads"], case["before"], case["after"], case["sinks"],
                                   kv_heads=case["kv_heads"])]
    if case["kind"] == "step":
        return [F.window_attention_step(s.q, s.k, s.v, s.lengths, case["heads"], case["before"], case["sinks"], kv_heads=case["kv_heads"])]
    return [F.type_cross_entropy(s.x, s.weight, s.target)]


def _spread(values, scales):
    """The values that 8 bits and their scales (nodes, groups) stand for."""
    n = values.shape[0]
    return (values.reshape(n, scales.shape[1], -1) * scales[:, :, None]).reshape(values.shape)


def _plain(s, leaves):
    """In float32 (64 bits where it matters); what trains gets float32 leaves, the rest is cast here and its results rounded."""
    case, dt = s.case, TYPES[s.case["type"]]
    if case["kind"] == "norm":
        x, *rest = leaves
        weight = rest[-1]
        if case["group"] >= 0:                              # values next to a border between two of 8 bits: 64 bits
            x, weight = x.double(), weight.double()
            total = x + rest[0].double() if case["residual"] else x
            n, count = total.shape[0], total[0].numel()
            groups = (total * weight).reshape(n, count // (case["group"] or count), -1)
            most = groups.abs().amax(-1, keepdim=True)
            ratio = groups * E4M3_MAX / torch.where(most > 0, most, torch.ones_like(most))     # the norm itself cancels
            grain = torch.ldexp(torch.ones_like(ratio), torch.frexp(ratio.abs()).exponent.clamp(min=-5) - 4)
            scale = most / E4M3_MAX / (total.square().mean((1, 2), keepdim=True) + EPS).sqrt()
            return [(torch.round(ratio / grain) * grain * scale).float().reshape(total.shape), total.to(dt)]
        total = x.float() + rest[0].float() if case["residual"] else x.float()
        y = total / (total.square().mean((1, 2), keepdim=True) + EPS).sqrt() * weight.float()
        return [y, total] if case["train"] else [y.to(dt), total.to(dt)]
    if case["kind"] == "rotary":
        angle = s.positions.double()[:, None] * s.frequencies
        outs = [_turn(t.float(), torch.cos(angle).float(), torch.sin(angle).float(), case["size"], case["interleaved"]) for t in leaves]
        return outs if case["train"] else [t.to(dt) for t in outs]
    if case["kind"] == "window":
        out = _plain_window(s, *(t.float() for t in leaves))
        return [out if case["train"] else out.to(dt)]
    if case["kind"] == "step":
        return [_plain_step(s).to(dt)]
    x, weight = (t.float() for t in leaves)
    logits = x @ weight.T
    counts = s.target >= 0
    top = logits.amax(1, keepdim=True).detach()
    losses = (logits - top).exp().sum(1).log() + top[:, 0] - logits.gather(1, s.target.clamp(min=0)[:, None])[:, 0]
    return [(losses * counts).sum() / counts.sum().clamp(min=1)]


def _turn(x, cos, sin, size, interleaved):
    n, d, channels = x.shape
    half = cos.shape[1]
    x = x.reshape(n, d, channels // size, size)
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    a, b = (turned[..., 0::2], turned[..., 1::2]) if interleaved else (turned[..., :half], turned[..., half:])
    cos, sin = cos[:, None, None], sin[:, None, None]
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turned, rest], -1).reshape(n, d, channels)


def _plain_window(s, q, k, v):
    """Blocks of 128 nodes against the keys that any of them may see, and each node against its chain's first ones."""
    case, block = s.case, 128
    n, d, _ = q.shape
    heads, kv, size, before, after, sinks = (case[x] for x in ("heads", "kv_heads", "size", "before", "after", "sinks"))
    before = min(before, n)
    after = min(after, n)
    rows = lambda t, h: t.view(n, d, h, size).transpose(1, 2).reshape(n, h, d * size)  # noqa: E731
    q, k, v = rows(q, heads), rows(k, kv), rows(v, kv)
    blocks = (n + block - 1) // block
    i = (torch.arange(blocks * block, device=DEV)).clamp(max=n - 1)
    graph = torch.searchsorted(s.ptr, i, right=True) - 1
    first, end = s.ptr[graph], s.ptr[graph + 1]
    j = torch.arange(blocks, device=DEV)[:, None] * block + torch.arange(-before, block + after, device=DEV)
    at = j.clamp(0, n - 1)
    place = i.view(blocks, block, 1)
    seen = ((j[:, None] >= torch.maximum(first.view(blocks, block, 1), place - before)) & (j[:, None] < end.view(blocks, block, 1))
            & (j[:, None] <= place + after))
    far = first[:, None] + torch.arange(sinks, device=DEV)
    far_seen = (far < (i - before)[:, None]).view(blocks, block, sinks)
    far = far.clamp(max=n - 1)
    mine = q[i].view(blocks, block, kv, heads // kv, d * size)
    keys, values = k[at], v[at]
    far_keys, far_values = (t[far].view(blocks, block, sinks, kv, d * size) for t in (k, v))
    # (blocks, kv heads, heads of each, rows, keys)
    score = torch.cat([torch.einsum("brkgc,bjkc->bkgrj", mine, keys).masked_fill(~seen[:, None, None], -torch.inf),
                       torch.einsum("brkgc,brjkc->bkgrj", mine, far_keys).masked_fill(~far_seen[:, None, None], -torch.inf)],
                      -1) / math.sqrt(d * size)
    weight = (score - score.amax(-1, keepdim=True).detach()).exp()
    weight = weight / weight.sum(-1, keepdim=True)
    split = j.shape[1]
    out = (torch.einsum("bkgrj,bjkc->brkgc", weight[..., :split], values)
           + torch.einsum("bkgrj,brjkc->brkgc", weight[..., split:], far_values))
    return out.reshape(blocks * block, heads, d, size)[:n].transpose(1, 2).reshape(n, d, heads * size)


def _plain_step(s):
    case = s.case
    graphs, d, _ = s.q.shape
    heads, kv, size = case["heads"], case["kv_heads"], case["size"]
    j = torch.arange(case["capacity"], device=DEV)
    last = s.lengths[:, None] - 1
    seen = (j <= last) & ((j >= last - case["before"]) | (j < case["sinks"]))
    q = s.q.float().view(graphs, d, kv, heads // kv, size)
    k, v = (t.float().view(graphs, -1, d, kv, size) for t in (s.k, s.v))
    score = torch.einsum("gdkhc,gjdkc->gkhj", q, k) / math.sqrt(d * size)
    score = score.masked_fill(~seen[:, None, None], -torch.inf)
    weight = (score - score.amax(-1, keepdim=True)).exp()
    weight = weight / weight.sum(-1, keepdim=True)
    return torch.einsum("gkhj,gjdkc->gdkhc", weight, v).reshape(graphs, d, heads * size)


def work(case):
    size, kind, train = 4 if case["type"] == "f32" else 2, case["kind"], case["train"]
    if kind == "norm":
        n, c = case["rows"], case["channels"]
        values = n * case["comps"] * c
        ins, outs = 1 + case["residual"], 1 + case["residual"]       # without a residual the sum is the input
        if case["group"] >= 0:
            return {"bytes": values * (ins * size + 1 + case["residual"] * size) + 4 * n * max(1, case["comps"] * c // (case["group"] or c * case["comps"])),
                    "flops": 8 * values}
        # backward: both gradients that come in, the sum, the gradient that goes out (one for x and the residual)
        return {"bytes": values * size * (ins + outs + (4 if train else 0)) + c * size, "flops": values * (16 if train else 5)}
    if kind == "rotary":
        values = case["rows"] * case["comps"] * (case["heads"] + case["kv_heads"]) * case["size"]
        return {"bytes": values * size * (4 if train else 2) + case["rows"] * 8, "flops": values * 3 * (2 if train else 1)}
    width, kv_width = (case.get("comps", 1) * case.get(h, 0) * case.get("size", 0) for h in ("heads", "kv_heads"))
    if kind == "window":
        sizes = _sizes(case)
        counts = {x: sizes.count(x) for x in set(sizes)}
        pairs = sum(m * _seen(x, case["before"], case["after"], case["sinks"]) for x, m in counts.items())
        n = sum(sizes)
        return {"bytes": n * (width * 2 + kv_width * 2) * (2 if train else 1) * size, "flops": pairs * width * (14 if train else 4)}
    if kind == "step":
        keys = sum(min(x, case["before"] + 1 + case["sinks"]) for x in _lengths(case))
        return {"bytes": (keys * 2 * kv_width + case["graphs"] * 2 * width) * size, "flops": keys * width * 4}
    n, t, c = case["rows"] * (1 - case["ignored"]), case["types"], case["channels"]
    return {"bytes": (n + t) * c * (2 if train else 1) * size + case["rows"] * 8, "flops": 2 * n * t * c * (4 if train else 1)}


# ---- definitions in 64 bits -----------------------------------------------------------------------------------------------------


def _exact_norm(s):
    case = s.case
    x = s.x.detach().double()
    h = x if s.residual is None else x + s.residual.detach().double()
    w = s.weight.detach().double()
    n = h.shape[0]
    count = h[0].numel()
    r = torch.rsqrt(torch.einsum("ndc,ndc->n", h, h) / count + EPS).view(n, 1, 1)
    unit = h * r
    y = unit * w
    if case["group"] >= 0:
        cut = (h * w).view(n, -1, case["group"] or count)
        largest = cut.abs().max(-1, keepdim=True).values
        ratio = torch.nan_to_num(cut * E4M3_MAX / largest, nan=0.0)
        # the nearest of 8 bits: three bits behind the leading one, not below 2^-9
        grain = torch.exp2(torch.floor(torch.log2(ratio.abs().clamp(min=2.0 ** -6))) - 3)
        return [(torch.round(ratio / grain) * grain * (largest * r / E4M3_MAX)).view_as(y), h]
    if not case["train"]:
        return [y, h]
    g, gh = (c.double() for c in s.cots)
    gw = g * w
    dh = gh + r * (gw - unit * ((gw * unit).sum((1, 2)) / count).view(n, 1, 1))
    return [y, h, dh, *([dh] if s.residual is not None else []), torch.einsum("ndc,ndc->c", g, unit)]


def _exact_rotary(s):
    case = s.case
    theta = torch.outer(s.positions.double(), s.frequencies)
    phase = torch.polar(torch.ones_like(theta), theta)[:, None, None]

    def turned(t, by):
        n, d, channels = t.shape
        out = t.double().reshape(n, d, -1, case["size"]).clone()
        part = out[..., :case["rotated"]].unflatten(-1, (-1, 2) if case["interleaved"] else (2, -1))
        if not case["interleaved"]:
            part = part.transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(part.contiguous()) * by)
        out[..., :case["rotated"]] = (z if case["interleaved"] else z.transpose(-1, -2)).flatten(-2)
        return out.view(n, d, channels)

    outs = [turned(t.detach(), phase) for t in (s.q, s.k)]
    return outs + [turned(c, phase.conj()) for c in s.cots] if case["train"] else outs


def _exact_window(s):
    case = s.case
    n, d, _ = s.q.shape
    heads, kv, size, before, after, sinks = (case[x] for x in ("heads", "kv_heads", "size", "before", "after", "sinks"))
    pick = lambda t, h: t.detach().double().view(n, d, -1, size)[:, :, h].reshape(n, d * size)  # noqa: E731
    full = lambda like: torch.zeros(n, d, like.shape[2] // size, size, dtype=torch.float64, device=DEV)  # noqa: E731
    out, gq, gk, gv = full(s.q), full(s.q), full(s.k), full(s.k)
    scale, ends = (d * size) ** -0.5, s.ptr.tolist()
    for h in range(heads):
        q, k, v = pick(s.q, h), pick(s.k, h // (heads // kv)), pick(s.v, h // (heads // kv))
        g = pick(s.cots[0], h) if case["train"] else None
        o, dq, dk, dv = (torch.zeros_like(q) for _ in range(4))
        for lo, hi in zip(ends[:-1], ends[1:]):
            for r0 in range(lo, hi, 2048):
                r1 = min(hi, r0 + 2048)
                j0 = max(lo, r0 - before)
                cols = torch.cat([torch.arange(lo, min(j0, lo + sinks), device=DEV), torch.arange(j0, min(hi, r1 + after), device=DEV)])
                i, j = torch.arange(r0, r1, device=DEV)[:, None], cols[None]
                hidden = (j > i + after) | ((j < i - before) & (j >= lo + sinks))
                z = torch.where(hidden, -torch.inf, scale * q[r0:r1] @ k[cols].T)
                p = torch.softmax(z, 1)
                o[r0:r1] = p @ v[cols]
                if g is None:
                    continue
                ds = p * (g[r0:r1] @ v[cols].T - (g[r0:r1] * o[r0:r1]).sum(1, keepdim=True)) * scale
                dq[r0:r1] = ds @ k[cols]
                dk.index_add_(0, cols, ds.T @ q[r0:r1])
                dv.index_add_(0, cols, p.T @ g[r0:r1])
        put = lambda t: t.view(n, d, size)  # noqa: E731
        out[:, :, h], gq[:, :, h] = put(o), put(dq)
        gk[:, :, h // (heads // kv)] += put(dk)
        gv[:, :, h // (heads // kv)] += put(dv)
    results = [out, gq, gk, gv] if case["train"] else [out]
    return [t.reshape(n, d, -1) for t in results]


def _exact_step(s):
    case = s.case
    graphs, d, _ = s.q.shape
    heads, kv, size = case["heads"], case["kv_heads"], case["size"]
    out = torch.zeros(graphs, d, heads, size, dtype=torch.float64, device=DEV)
    for g, length in enumerate(s.lengths.tolist()):
        low = max(0, length - 1 - case["before"])
        cols = list(range(min(low, case["sinks"]))) + list(range(low, length))
        k, v = (t[g, cols].double().view(len(cols), d, kv, 1, size).expand(-1, -1, -1, heads // kv, -1).reshape(len(cols), d, heads, size)
                for t in (s.k, s.v))
        z = torch.einsum("dhc,jdhc->hj", s.q[g].double().view(d, heads, size), k) * (d * size) ** -0.5
        out[g] = torch.einsum("hj,jdhc->dhc", torch.softmax(z, 1), v)
    return [out.view(graphs, d, heads * size)]


def _exact_loss(s):
    x, w = s.x.detach().double(), s.weight.detach().double()
    rows = (s.target >= 0).nonzero()[:, 0]
    count = max(1, rows.numel())
    dx, dw, loss = torch.zeros_like(x), torch.zeros_like(w), torch.zeros((), dtype=torch.float64, device=DEV)
    for part in rows.split(2048):
        log_p = torch.log_softmax(torch.einsum("nc,tc->nt", x[part], w), 1)
        at = (torch.arange(part.numel(), device=DEV), s.target[part])
        loss -= log_p[at].sum() / count
        if s.case["train"]:
            g = log_p.exp_()
            g[at] -= 1.0
            g /= count
            dx[part] = g @ w
            dw += g.T @ x[part]
    return [loss, dx, dw] if s.case["train"] else [loss]


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "rotary": _exact_rotary, "window": _exact_window, "step": _exact_step, "loss": _exact_loss}[case["kind"]](s)
