"""Tree attention where many queries share a key head, capped and biased, for every type: a node's
result is as exact in a large tree as in a small one.

Tolerance, for every number of columns. Products of bfloat16 numbers (codes hold 8 bits, float32
queries are three bfloat16 numbers to 2^-26) are exact in float32 and a score sums D of them, plus a few
steps of its scaling: it is off by at most
    delta = (D + 4) 2^-24 scale sum |q_f k_f| + 2^-21 (|raw| + |s| + cap + bias),
a probability by 2 max(delta) of itself. The sums over T tokens run over 64 at a time, then over blocks,
wavefronts and splits: at most T / 64 + 96 roundings of 2^-24, twice (numerator and denominator).
Results of bfloat16 take probabilities to 2^-16 and are rounded once, by half a step; float32 ones take
probabilities to 2^-24."""

from __future__ import annotations

import math

import pytest
import torch

import draft_reference as plain
from local_ai_training.drafts import draft_tree, tree_attention
from local_ai_training.int8_cache import int8_kv, int8_kv_append, int8_kv_read

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def rows(cuda, b, h, n, d, seed, dtype, std=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(b, h, n, d, generator=gen) * std).to(dtype).to(cuda)


def check(cuda, d, nodes, group, dtype, out, cap=0.0, biased=False, start=(290, 131), scale=None):
    b, h = len(start), 2
    cache = int8_kv(b, h, 300, d, cuda)
    int8_kv_append(cache, rows(cuda, b, h, 300, d, 1, BF16), rows(cuda, b, h, 300, d, 2, BF16),
                   torch.tensor([0], device=cuda))
    q = rows(cuda, b, h * group, nodes, d, 3, dtype, 1.5)
    k, v = (rows(cuda, b, h, nodes, d, s, dtype) for s in (4, 5))
    slopes = torch.exp2(-torch.arange(1, h * group + 1, dtype=F32)) if biased else None
    parents = [plain.random_parents(nodes, s) for s in range(b)]
    got = tree_attention(q, k, v, cache, torch.tensor(start, device=cuda),
                         draft_tree(parents, cuda), softcap=cap or None,
                         slopes=slopes.to(cuda) if biased else None, scale=scale, out_dtype=out)
    assert got.dtype == out
    keys, values = (t.double().cpu() for t in int8_kv_read(cache))
    few = 2.0**-16 if out == BF16 else 2.0**-24
    for s, past in enumerate(start):
        args = (t[s].double().cpu() for t in (q, k, v))
        want, size, delta = plain.tree_attention(
            *args, keys[s, :, :past], values[s, :, :past], past, parents[s], cap,
            slopes.double() if biased else None, scale or 1.0 / math.sqrt(d))
        bound = ((2 * delta + 2 * (past / 64 + 96) * 2.0**-24 + few) * size
                 + torch.finfo(out).eps / 2 * want.abs())
        worst = ((got[s].double().cpu() - want).abs() - bound).max().item()
        assert worst <= 0.0, (s, worst)


@pytest.mark.parametrize("cap,biased", [(0.0, False), (2.0, False), (50.0, False), (0.0, True),
                                        (20.0, True)])
@pytest.mark.parametrize("d,nodes,group", [(64, 17, 2), (64, 40, 8), (128, 33, 1), (128, 12, 4),
                                           (256, 34, 1)])
def test_many_columns(cuda, d, nodes, group, cap, biased):
    """More than 32 queries a key head, bfloat16 results of bfloat16 queries."""
    print(f"columns D={d} N={nodes} G={group} cap={cap} bias={biased}", flush=True)
    check(cuda, d, nodes, group, BF16, BF16, cap, biased)


@pytest.mark.parametrize("cap,biased", [(2.0, False), (30.0, False), (0.0, True), (20.0, True)])
@pytest.mark.parametrize("out", [BF16, F32])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d,nodes,group", [(64, 9, 2), (64, 21, 2), (128, 9, 2), (256, 9, 1)])
def test_modified_scores_of_every_type(cuda, d, nodes, group, dtype, out, cap, biased):
    print(f"scores D={d} N={nodes} {dtype} {out} cap={cap} bias={biased}", flush=True)
    check(cuda, d, nodes, group, dtype, out, cap, biased, scale=0.3)
