"""Attention within windows of chains in float64, and how far a kernel may be from it.

Bounds count roundings.  ``u``: half a step of the features' type (results, and of bfloat16 the weights and score gradients of products);
``c``: what a float32 sum of at most 128 products loses in the tensor cores, of the sum of the products' absolute values.  float32 products are of TF32
pairs (2^-21 each) added eight at a time with truncation (16 steps of 2^-23), bfloat16 ones are exact, sixteen at a time (8 steps); long
sums over keys are bounded likewise, 16 or 8 steps a tile of at most 128 keys and one rounding a tile."""
import math

import torch

UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
SUM = {torch.float32: 2.0 ** -18, torch.bfloat16: 2.0 ** -19}


def heads_of(t, heads):
    """(N, components, channels) as (heads, N, values of a head)."""
    n, d, c = t.shape
    return t.detach().double().view(n, d, heads, c // heads).permute(2, 0, 1, 3).reshape(heads, n, -1)


def back(t, d):
    """The other way round."""
    heads, n, values = t.shape
    return t.view(heads, n, d, values // d).permute(1, 2, 0, 3).reshape(n, d, -1)


def seen(sizes, n, before, after, sinks, first=0):
    mask = torch.zeros(n, n, dtype=torch.bool)
    lo = first
    for size in sizes:
        i, j = torch.arange(size)[:, None], torch.arange(size)[None]
        mask[lo:lo + size, lo:lo + size] = (j <= i + after) & ((j >= i - before) | (j < sinks))
        lo += size
    return mask


def reference(q, k, v, g, mask, heads, kv_heads, scale):
    """Results (out, dq, dk, dv) and bounds of their errors, both (N, components, channels) float64."""
    u, c, d = UNIT[q.dtype], SUM[q.dtype], q.shape[1]
    group = heads // kv_heads
    spread = lambda t: t.repeat_interleave(group, 0)  # noqa: E731
    q, g = heads_of(q, heads), heads_of(g, heads)
    k, v = spread(heads_of(k, kv_heads)), spread(heads_of(v, kv_heads))
    scale = scale if scale is not None else 1 / math.sqrt(q.shape[2])
    mask = mask.to(q.device)
    t = lambda x: x.transpose(1, 2)  # noqa: E731
    none = ~mask.any(1)
    s = (scale * q @ t(k)).masked_fill(~mask, -math.inf)
    s = s - s.amax(2, keepdim=True).nan_to_num(neginf=0.0)
    p = s.exp()
    p = p / p.sum(2, keepdim=True).masked_fill(none[None, :, None], 1.0)
    out = p @ v
    dp, delta = g @ t(v), (g * out).sum(2, keepdim=True)
    ds = p * (dp - delta)
    dq, dk, dv = scale * ds @ k, scale * t(ds) @ q, t(p) @ g
    # scores to within es, so weights to within their share, the sum's, and a rounding for the product
    es = abs(scale) * c * q.abs() @ t(k.abs()) + 2.0 ** -21 * s.abs().masked_fill(~mask, 0.0)
    ep = p * (es + (p * es).sum(2, keepdim=True) + u + 2.0 ** -20)
    eout = ep @ v.abs() + c * (p @ v.abs()) + u * out.abs()
    edelta = (g.abs() * eout).sum(2, keepdim=True) + c * (g * out).abs().sum(2, keepdim=True)
    eds = ep * (dp - delta).abs() + p * (c * (g.abs() @ t(v.abs())) + edelta) + u * ds.abs()
    edq = abs(scale) * (eds + c * ds.abs()) @ k.abs() + u * dq.abs()
    edk = abs(scale) * t(eds + c * ds.abs()) @ q.abs()
    edv = t(ep + c * p) @ g.abs()
    folded = lambda x: x.view(kv_heads, group, *x.shape[1:]).sum(1)  # noqa: E731
    dk, dv, edk, edv = folded(dk), folded(dv), folded(edk), folded(edv)
    return [back(x, d) for x in (out, dq, dk, dv)], [back(x, d) for x in (eout, edq, edk + u * dk.abs(), edv + u * dv.abs())]
