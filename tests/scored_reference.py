"""Attention with modified scores in 64 bits, and the bounds its bf16 kernels are held to."""

from __future__ import annotations

import math

import torch

U = 2.0 ** -8   # half a bf16 step, relative to the value
W = 2.0 ** -12  # what float32 scores, exponentials and log-sum-exps move a probability by


def seen_keys(documents, prefix, b, s):
    """[B, S, S] bool from the definition, a position at a time (CPU lists)."""
    seen = torch.zeros(b, s, s, dtype=torch.bool)
    for r in range(b):
        ids = documents[r].tolist() if documents is not None else [0] * s
        marks = prefix[r].tolist() if prefix is not None else [False] * s
        low = 0
        while low < s:
            high = low
            while high < s and ids[high] == ids[low]:
                high += 1
            lead = low
            while lead < high and marks[lead]:
                lead += 1
            if ids[low] >= 0:
                for i in range(low, high):
                    seen[r, i, low:max(lead, i + 1)] = True
            low = high
    return seen


def layout(kind, b, s, seed=0):
    """(documents, prefix) of a mask kind: None, documents of several lengths with padding
    between and behind them, marked beginnings (some marks behind them), or both."""
    gen = torch.Generator().manual_seed(seed + s)
    documents = prefix = None
    if "documents" in kind:
        cuts = torch.rand(b, s, generator=gen) < 3.0 / max(s, 6)
        documents = cuts.cumsum(1)
        hole = torch.rand(b, s, generator=gen) < 0.5
        documents = torch.where((documents % 3 == 2) & hole[:, :1], -1 - (documents % 2), documents)
        documents[-1, (2 * s) // 3:] = -1
    if "prefix" in kind:
        prefix = torch.rand(b, s, generator=gen) < 0.1
        prefix[:, :s // 3] = True
        if documents is not None:
            prefix |= documents % 2 == 1
    return documents, prefix


def reference(q, k, v, g, seen, cap, slopes, scale):
    """float64 (o, dq, dk, dv, dslopes) and the bound on each element (any device).

    u is half a bf16 step, w what the float32 scores move a probability by. p and ds enter their
    products rounded (u), every bf16 result is rounded once (u). The kernels' o is off by
    Eo = (u + w) p |v| + u |o|, so delta = g . o by Ed = |g| . Eo; the float32 sums g . v and
    g . o by 2^-17 of their absolute sums. Gradients d of the modified scores are off by
    E = p (Ed + 2^-17 (|g| . |v| + |g| . |o|)) + w |d|, those of the plain ones by that times the
    tanh's slope t' plus w |d|. The slopes' gradient takes -delta only as a reference that
    cancels: each product p (dp - delta') (|i - j| - mean) is off by w of its absolute factors."""
    dt = torch.float64
    q, k, v, g = (t.detach().to(dt).contiguous() for t in (q, k, v, g))
    b, h, s, d = q.shape
    group = h // k.shape[1]
    kk, vv = (t.repeat_interleave(group, dim=1) for t in (k, v))

    def tr(t):
        return t.transpose(-1, -2).contiguous()

    def shared(t):
        return t.view(b, h // group, group, s, d).sum(2)

    at = torch.arange(s, device=q.device, dtype=dt)
    dist = (at[:, None] - at[None, :]).abs()
    seen = seen.to(q.device)[:, None]
    raw = q @ tr(kk) * scale
    t = torch.tanh(raw / cap) if cap else torch.zeros_like(raw)
    scores = cap * t if cap else raw
    if slopes is not None:
        scores = scores - slopes.detach().to(q.device, dt)[:, None, None] * dist
    some = seen.any(-1, keepdim=True)
    p = torch.where(some, scores.masked_fill(~seen, -math.inf), 0.0).softmax(-1)
    p = p.masked_fill(~seen, 0.0)
    o = p @ vv
    eo = (U + W) * (p @ vv.abs()) + U * o.abs()
    delta = (g * o).sum(-1, keepdim=True)
    ed = (g.abs() * eo).sum(-1, keepdim=True)
    dp = g @ tr(vv)
    sums = 2.0 ** -17 * (g.abs() @ tr(vv.abs()) + (g * o).abs().sum(-1, keepdim=True))
    grad = p * (dp - delta)
    e = p * (ed + sums) + W * grad.abs()
    slack = 1.0 - t * t
    ds, es = grad * slack, e * slack + W * grad.abs()
    es = es + U * ds.abs()
    out = [(o, eo), (scale * ds @ kk, scale * es @ kk.abs()),
           (shared(scale * tr(ds) @ q), shared(scale * tr(es) @ q.abs())),
           (shared(tr(p) @ g), shared((U + W) * tr(p) @ g.abs()))]
    out = [out[0]] + [(x, bound + U * x.abs()) for x, bound in out[1:]]
    mean = (p * dist).sum(-1, keepdim=True)
    spread = p * ((dp - delta).abs() + ed) * (dist + mean) * 2.0 * W + p * sums * (dist + mean)
    out.append((-(grad * dist).sum((0, 2, 3)),
                spread.sum((0, 2, 3)) + 2.0 ** -24 * (grad * dist).sum((0, 2, 3)).abs()))
    return out
