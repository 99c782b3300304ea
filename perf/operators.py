"""The operators of a transformer layer over packed graphs, and what they are timed on: the calls that a user makes, their plain
forms in elementary torch operations, and their definitions in 64 bits.

attention   ``graph_attention``: the nodes of each graph of a batch attend to the nodes of the same graph; a head's score is the inner
            product over all components of its channels, capped by a tanh where a cap is given, less a slope times the distance of
            the two nodes where positions are given
gated       ``gated_linear``: both projections of a gated feed-forward block, the activation and the product
embedding   ``type_embedding``: rows of a table by node or edge type, scaled, and the table's gradient
"""
from __future__ import annotations

import math
import random
from types import SimpleNamespace

import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # A small training batch of molecules, 32 graphs of 30 atoms: launches and latency count.
        dict(name="attention_f32_32x30", kind="attention", type="f32", graphs=32, low=30, high=30, comps=1, channels=128, heads=4,
             bias=True, cap=0.0, train=True),
        # A large training batch of ragged molecules, 5 to 60 atoms each.
        dict(name="attention_bf16_molecules", kind="attention", type="bf16", graphs=2000, low=5, high=60, comps=1, channels=256,
             heads=8, bias=True, cap=20.0, train=True),
        # Equivariant features 0e+1o+2e: nine components of 64 channels, clusters of 40 to 250 atoms.
        dict(name="attention_f32_equivariant", kind="attention", type="f32", graphs=48, low=40, high=250, comps=9, channels=64,
             heads=8, bias=True, cap=0.0, train=True),
        # One periodic box or protein as a single graph: the quadratic work counts.
        dict(name="attention_bf16_one_graph", kind="attention", type="bf16", graphs=1, low=5001, high=5001, comps=1, channels=512,
             heads=8, bias=True, cap=30.0, train=True),
        # Scoring structures of very different sizes, some of a single atom or none: forward only.
        dict(name="attention_bf16_infer_ragged", kind="attention", type="bf16", graphs=16, low=0, high=2000, comps=1, channels=256,
             heads=8, bias=True, cap=0.0, train=False),
        # Feed-forward of the small batch of molecules.
        dict(name="gated_f32_960", kind="gated", type="f32", rows=960, channels=128, hidden=256, act="silu", train=True),
        # Feed-forward of a large training step.
        dict(name="gated_bf16_100k", kind="gated", type="bf16", rows=100_000, channels=256, hidden=1024, act="silu", train=True),
        # Narrow layer, ragged sizes, float32.
        dict(name="gated_f32_50021", kind="gated", type="f32", rows=50_021, channels=64, hidden=200, act="gelu", train=True),
        # A wide block at inference.
        dict(name="gated_bf16_infer_wide", kind="gated", type="bf16", rows=8_192, channels=1024, hidden=4096, act="silu", train=False),
        # Atom types of the small batch of molecules.
        dict(name="embedding_f32_960", kind="embedding", type="f32", rows=960, types=119, channels=128, skew=1.0, train=True),
        # Atom types of a large training step: few types, most atoms of the first ones.
        dict(name="embedding_f32_100k", kind="embedding", type="f32", rows=100_000, types=119, channels=64, skew=1.0, train=True),
        # Pairs of atom types on the edges of the large step: many types, ragged count.
        dict(name="embedding_bf16_pairs_2m", kind="embedding", type="bf16", rows=1_998_931, types=14_161, channels=32, skew=0.7,
             train=True),
    ]


def _log(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return min(hi, n | 1) if rng.random() < 0.5 else n


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "gated", "gated", "embedding"])
    kind_type = rng.choice(["f32", "bf16"])
    train = rng.random() < 0.75
    if kind == "attention":
        comps = rng.choice([1, 1, 1, 4, 9])
        heads = rng.choice([1, 2, 4, 8, 8])
        size = rng.choice([16, 32, 64, 128] if comps == 1 else [8, 16] if comps == 4 else [8])
        high = _log(rng, 8, 4000)
        low = rng.choice([0, 1, high // 8, high // 2, high])
        area = 2.0e8 / (heads * (4 if kind_type == "f32" else 1))          # a call costs no more than the largest listed one
        graphs = max(1, min(_log(rng, 1, 2000), int(area / high ** 2), int(6.0e7 / (high * comps * heads * size))))
        high = min(high, int(math.sqrt(area)))
        return dict(kind=kind, type=kind_type, graphs=graphs, low=min(low, high), high=high, comps=comps, channels=heads * size,
                    heads=heads, bias=rng.random() < 0.7, cap=rng.choice([0.0, 0.0, 20.0, 50.0]), train=train)
    if kind == "gated":
        channels = rng.choice([rng.randint(16, 128), 64, 128, 256, 512, _log(rng, 64, 1024)])
        hidden = channels * rng.choice([1, 2, 3, 4]) + rng.choice([0, 0, 8, 5])
        most = 2.6e10 / (channels * hidden) / (4 if kind_type == "f32" else 1)
        return dict(kind=kind, type=kind_type, rows=max(1, min(_log(rng, 1, 100_000), int(most))), channels=channels, hidden=hidden,
                    act=rng.choice(["silu", "silu", "gelu", "relu", "sigmoid"]), train=train)
    return dict(kind=kind, type=kind_type, rows=_log(rng, 1, 1_900_000), types=_log(rng, 2, 15_000),
                channels=rng.choice([16, 32, 32, 48, 31]), skew=rng.choice([0.0, 0.7, 1.0]), train=train)


def _sizes(case):
    """Nodes of each graph, ascending counts shuffled by the case's own numbers (not by the seed: `work` counts them too)."""
    low, high, graphs = case["low"], case["high"], case["graphs"]
    sizes = [low + (high - low) * i // max(1, graphs - 1) for i in range(graphs)] if graphs > 1 else [high]
    random.Random(graphs * 7919 + high).shuffle(sizes)
    return sizes


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = TYPES[case["type"]]
    rand = lambda *shape: torch.randn(*shape, device=DEV, generator=g)  # noqa: E731
    s = SimpleNamespace(case=case)
    if case["kind"] == "attention":
        sizes = _sizes(case)
        n, d, c, heads = sum(sizes), case["comps"], case["channels"], case["heads"]
        s.longest = max(sizes)
        s.ptr = torch.tensor([0] + sizes, device=DEV).cumsum(0)
        s.q, s.k, s.v, s.cot = (rand(n, d, c).to(dt) for _ in range(4))
        s.scale = 1.5 / math.sqrt(d * c // heads)
        # atoms at the density of a condensed phase, graphs in boxes of their own; head slopes from 1 to 1/16 per length unit
        box = (torch.tensor(sizes, device=DEV).double() * 10.0).pow(1 / 3).float().repeat_interleave(torch.tensor(sizes, device=DEV))
        s.pos = torch.rand(n, 3, device=DEV, generator=g) * box[:, None] if case["bias"] else None
        s.slope = (2.0 ** -torch.linspace(0, 4, heads, device=DEV) * (1 + 0.1 * rand(heads))) if case["bias"] else None
        if own:
            from equitorch_b200.graph import PackedGraphs
            s.graphs = PackedGraphs(s.ptr, n)
        s.leaves = [t for t in (s.q, s.k, s.v, s.slope, s.pos) if t is not None]
    elif case["kind"] == "gated":
        c, f = case["channels"], case["hidden"]
        s.x, s.weight = rand(case["rows"], c).to(dt), (rand(2, c, f) / math.sqrt(c)).to(dt)
        s.cot = rand(case["rows"], f).to(dt) if case["train"] else None
        s.leaves = [s.x, s.weight]
    else:
        t = case["types"]
        # type frequencies fall off as rank ** -skew, the types in no order
        prob = torch.arange(1, t + 1, device=DEV, dtype=torch.float32).pow(-case["skew"])
        edges = (prob.double().cumsum(0) / prob.double().sum()).float()
        rank = torch.searchsorted(edges, torch.rand(case["rows"], device=DEV, generator=g)).clamp_(max=t - 1)
        s.index = torch.randperm(t, device=DEV, generator=g)[rank]
        s.weight, s.scale = rand(t, case["channels"]).to(dt), 1 / math.sqrt(2)
        s.cot = rand(case["rows"], case["channels"]).to(dt) if case["train"] else None
        s.leaves = [s.weight]
    if case["train"]:
        for leaf in s.leaves:
            leaf.requires_grad_(True)
    return s


def run(s):
    if own:
        out = _call(s)
        return [out, *torch.autograd.grad(out, s.leaves, s.cot)] if s.case["train"] else out
    wide = [t.detach().float().requires_grad_(s.case["train"]) for t in s.leaves]
    out = _plain(s, wide)
    grads = torch.autograd.grad(out, wide, s.cot.float()) if s.case["train"] else []
    out = out.detach().to(TYPES[s.case["type"]])
    return [out, *(a.to(b.dtype) for a, b in zip(grads, s.leaves))] if s.case["train"] else out


def _call(s):
    from equitorch_b200.nn import functional as F
    if s.case["kind"] == "attention":
        return F.graph_attention(s.q, s.k, s.v, s.graphs, s.case["heads"], scale=s.scale, cap=s.case["cap"] or None, pos=s.pos,
                                 slope=s.slope)
    if s.case["kind"] == "gated":
        return F.gated_linear(s.x, s.weight, s.case["act"])
    return F.type_embedding(s.index, s.weight, s.scale)


ACTIVATIONS = {
    "silu": lambda x: x / (1 + torch.exp(-x)),
    "gelu": lambda x: 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5))),
    "relu": lambda x: x.clamp(min=0),
    "sigmoid": lambda x: 1 / (1 + torch.exp(-x)),
}


def _plain(s, leaves):
    case = s.case
    if case["kind"] == "embedding":
        return leaves[0][s.index] * s.scale
    if case["kind"] == "gated":
        x, w = leaves
        return ACTIVATIONS[case["act"]](x @ w[0]) * (x @ w[1])
    q, k, v, *rest = leaves
    (n, d, c), heads, longest = q.shape, case["heads"], s.longest
    # every graph padded to the longest: places (graphs, longest) and which of them hold a node
    places = s.ptr[:-1, None] + torch.arange(longest, device=DEV)
    there = places < s.ptr[1:, None]
    at = places.clamp(max=n - 1)
    rows = lambda t: t.view(n, d, heads, c // heads).transpose(1, 2).reshape(n, heads, -1)[at].transpose(1, 2)  # noqa: E731
    score = rows(q) @ rows(k).transpose(-1, -2) * s.scale
    if case["cap"]:
        score = case["cap"] * torch.tanh(score / case["cap"])
    if case["bias"]:
        slope, pos = rest
        diff = pos[at][:, :, None] - pos[at][:, None]
        square = diff.square().sum(-1)
        dist = torch.where(square > 0, torch.where(square > 0, square, torch.ones_like(square)).sqrt(), torch.zeros_like(square))
        score = score - slope[:, None, None] * dist[:, None]
    score = score.masked_fill(~there[:, None, None], -torch.inf)
    score = score - torch.where(there.any(1)[:, None, None, None], score.amax(-1, keepdim=True), torch.zeros_like(score[..., :1])).detach()
    weight = torch.exp(score)
    weight = weight / weight.sum(-1, keepdim=True).clamp(min=1e-30)
    out = (weight @ rows(v)).transpose(1, 2)[there]
    return out.view(n, heads, d, c // heads).transpose(1, 2).reshape(n, d, c)


def work(case):
    size = 4 if case["type"] == "f32" else 2
    times = 3 if case["train"] else 1
    if case["kind"] == "attention":
        sizes = _sizes(case)
        n, d, c, heads = sum(sizes), case["comps"], case["channels"], case["heads"]
        values = n * d * c * (8 if case["train"] else 4) * size
        return {"bytes": values + (n * 24 if case["bias"] else 0),
                "flops": sum(x * x for x in sizes) * d * c * (14 if case["train"] else 4)}
    if case["kind"] == "gated":
        n, c, f = case["rows"], case["channels"], case["hidden"]
        return {"bytes": (n * (c + f) + 2 * c * f) * (2 if case["train"] else 1) * size, "flops": 4 * n * c * f * times}
    n, t, c = case["rows"], case["types"], case["channels"]
    return {"bytes": n * 8 + (n * c + t * c) * (2 if case["train"] else 1) * size, "flops": n * c * (2 if case["train"] else 1)}


# ---- definitions in 64 bits -----------------------------------------------------------------------------------------------------


def _exact_attention(s, train):
    case = s.case
    n, d, c = s.q.shape
    heads = case["heads"]
    size = c // heads
    q, k, v, cot = (t.detach().double().reshape(n, d, heads, size) for t in (s.q, s.k, s.v, s.cot))
    out, gq, gk, gv = (torch.zeros_like(q) for _ in range(4))
    gslope = torch.zeros(heads, dtype=torch.float64, device=DEV)
    gpos = torch.zeros(n, 3, dtype=torch.float64, device=DEV)
    ends = s.ptr.tolist()
    for lo, hi in zip(ends[:-1], ends[1:]):
        if hi == lo:
            continue
        if case["bias"]:
            p = s.pos.detach().double()[lo:hi]
            diff = p[:, None] - p[None]
            r = (diff * diff).sum(-1).sqrt()
            unit = diff / torch.where(r > 0, r, torch.ones_like(r))[..., None]
        for h in range(heads):
            a, b, w, g = (t[lo:hi, :, h].reshape(hi - lo, d * size) for t in (q, k, v, cot))
            z = s.scale * torch.einsum("id,jd->ij", a, b)
            t = torch.tanh(z / case["cap"]) if case["cap"] else None
            e = z if t is None else case["cap"] * t
            if case["bias"]:
                e = e - s.slope.detach().double()[h] * r
            p_ij = torch.softmax(e, dim=1)
            o = p_ij @ w
            out[lo:hi, :, h] = o.view(-1, d, size)
            if not train:
                continue
            de = p_ij * (torch.einsum("id,jd->ij", g, w) - (o * g).sum(1, keepdim=True))
            dz = s.scale * (de if t is None else de * (1 - t * t))
            gv[lo:hi, :, h] = (p_ij.T @ g).view(-1, d, size)
            gq[lo:hi, :, h] = (dz @ b).view(-1, d, size)
            gk[lo:hi, :, h] = (dz.T @ a).view(-1, d, size)
            if case["bias"]:
                gslope[h] -= (de * r).sum()
                gpos[lo:hi] -= s.slope.detach().double()[h] * torch.einsum("ij,ijx->ix", de + de.T, unit)
    full = lambda t: t.reshape(n, d, c)  # noqa: E731
    if not train:
        return full(out)
    return [full(out), full(gq), full(gk), full(gv), *([gslope, gpos] if case["bias"] else [])]


def _exact_gated(s, train):
    x, w0, w1 = s.x.detach().double(), s.weight[0].detach().double(), s.weight[1].detach().double()
    a, u = torch.mm(x, w0), torch.mm(x, w1)
    sig = torch.sigmoid(a)
    if s.case["act"] == "silu":
        y, dy = a * sig, sig * (1 + a * (1 - sig))
    elif s.case["act"] == "sigmoid":
        y, dy = sig, sig * (1 - sig)
    elif s.case["act"] == "relu":
        y, dy = torch.relu(a), (a > 0).double()
    else:
        half = torch.special.ndtr(a)
        y, dy = a * half, half + a * torch.exp(-0.5 * a * a) / math.sqrt(2 * math.pi)
    if not train:
        return y * u
    g = s.cot.double()
    da, du = g * u * dy, g * y
    return [y * u, torch.mm(da, w0.T) + torch.mm(du, w1.T), torch.stack([torch.mm(x.T, da), torch.mm(x.T, du)])]


def _exact_embedding(s, train):
    table = s.weight.detach().double()
    out = torch.index_select(table, 0, s.index).mul_(s.scale)
    if not train:
        return out
    return [out, torch.zeros_like(table).index_add_(0, s.index, s.cot.double()).mul_(s.scale)]


def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "gated": _exact_gated, "embedding": _exact_embedding}[case["kind"]](s, case["train"])
