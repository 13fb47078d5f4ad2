"""Plain forms of drafted trees in 64 bits, from the definitions and one node at a time."""

from __future__ import annotations

import math
import random

import torch


def random_parents(nodes: int, seed: int, reach: int = 6) -> list[int]:
    rng = random.Random(seed)
    return [-1] + [rng.randint(max(0, i - reach), i - 1) for i in range(1, nodes)]


def way_of(parents: list[int], node: int) -> list[int]:
    """From the root to the node."""
    way = []
    while node >= 0:
        way.append(node)
        node = parents[node]
    return way[::-1]


def tree_attention(q, k, v, keys, values, start, parents, cap, slopes, scale):
    """One sequence on the CPU: q [Hq, N, D], k, v [H, N, D], keys, values [H, start, D], float64.
    Returns the result and, for its tolerance, sum p |v| and the largest error of a score by the
    roundings of its sums (see test_gpu_drafts.py)."""
    hq, n, d = q.shape
    group = hq // k.shape[0]
    out, size, worst = (torch.zeros(hq, n, x) for x in (d, d, 1))
    out, size, worst = out.double(), size.double(), worst.double()
    for i in range(n):
        way = way_of(parents, i)
        kk = torch.cat([keys, k[:, way]], dim=1).repeat_interleave(group, dim=0)
        vv = torch.cat([values, v[:, way]], dim=1).repeat_interleave(group, dim=0)
        place = torch.cat([torch.arange(start), start + torch.arange(len(way))]).double()
        distance = start + len(way) - 1 - place
        s = (kk * q[:, i, None]).sum(-1) * scale
        products = (kk * q[:, i, None]).abs().sum(-1) * scale
        raw = s.abs()
        if cap:
            s = cap * torch.tanh(s / cap)
        bias = slopes[:, None] * distance if slopes is not None else torch.zeros_like(s)
        s = s - bias
        p = s.softmax(-1)
        out[:, i] = (p[..., None] * vv).sum(1)
        size[:, i] = (p[..., None] * vv.abs()).sum(1)
        delta = (d + 4) * 2.0**-24 * products + 2.0**-21 * (raw + s.abs() + cap + bias.abs())
        worst[:, i, 0] = delta.amax(-1)
    return out, size, worst


def distribution(row, temperature, top_k):
    x = row.double()
    if top_k and top_k < len(x):
        least = sorted(x.tolist())[-top_k]
        x = torch.where(x < least, -math.inf, x)
    x = x / temperature
    e = torch.exp(x - x.max())
    return e / e.sum()


def verify(logits, tokens, parents, uniforms, drafts, temperature, top_k):
    """One sequence on the CPU: logits [N, V]. Returns the way, the next token, and how near the
    nearest decision came to its border."""
    way, near = [0], math.inf
    while True:
        node = way[-1]
        children = [i for i in range(len(parents)) if parents[i] == node]
        if temperature == 0.0:
            best = int((logits[node] == logits[node].max()).nonzero()[0])
            match = [i for i in children if int(tokens[i]) == best]
            if not match:
                return way, best, near
            way.append(match[0])
            continue
        p = distribution(logits[node], temperature, top_k)
        q = distribution(drafts[node], temperature, top_k) if drafts is not None else None
        size = p  # what p's roundings are relative to: p before anything was taken from it
        for i in children:
            x = int(tokens[i])
            chance = float(q[x]) if q is not None else 1.0
            if float(p[x]) > 0.0:  # (a zero is one in any order of the sums)
                drawn = float(uniforms[i]) * chance
                near = min(near, abs(drawn - float(p[x])) / max(drawn, float(size[x])))
            if float(uniforms[i]) * chance < float(p[x]):
                way.append(i)
                break
            left = (p - q).clamp(min=0.0) if q is not None else p * (torch.arange(len(p)) != x)
            if float(left.sum()) > 2.0**-40:
                p, size = left / left.sum(), size / left.sum()
        if way[-1] == node:
            sums = torch.cumsum(p, 0)
            bound = float(uniforms[0]) * float(sums[-1])
            if bound > 0.0:
                near = min(near, float((sums - bound).abs().min()))
            return way, int((sums > bound).nonzero()[0]), near
