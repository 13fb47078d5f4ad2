"""Attention over the 8-bit cache where numbers of very different size meet, against 64 bits over
the values the codes stand for: a feature far above a query's others.

Tolerance. A query is a fixed-point number of 127 256^2 steps, off by at most half a step, 2^-23.98
of its row's largest feature; its digits' integer sums are exact, and joining them in float32 takes
2^-9 of a step times the codes' sum and 2^-24 of the score. So a score is off by at most
    delta = 2^-23 scale max|q| sum|k| + 2^-21 |s|
(twice the half step, and the roundings of scales, exponentials' arguments and sums), a probability
by 2 max(delta) of itself and 2^-20 for exponentials and sums. Fixed-point probabilities are off by
half a step of their block's largest, over 64 tokens 2^(5 - r) of the values' largest with r = 23 bits
for float32 results and 15 for bfloat16 ones, which are rounded once, by 2^-8 of themselves."""

from __future__ import annotations

import math

import pytest
import torch

from local_ai_training.int8_cache import int8_kv, int8_kv_append, int8_kv_attention, int8_kv_read

pytestmark = pytest.mark.gpu


def filled(cuda, k, v):
    cache = int8_kv(k.shape[0], k.shape[1], k.shape[2], k.shape[3], cuda)
    int8_kv_append(cache, k, v, torch.zeros(1, dtype=torch.int64, device=cuda))
    return cache


def scores_of(q, cache, n):
    """float64 (scores, values, bound on a score) of the last of n positions."""
    keys, values = (t.double() for t in int8_kv_read(cache, 0, n))
    scale = 1.0 / math.sqrt(q.shape[-1])
    x = q.double()
    s = x @ keys.transpose(2, 3).contiguous() * scale
    size = scale * x.abs().amax(-1, keepdim=True) * keys.abs().sum(-1)[:, :, None]
    return s, values, 2.0**-23 * size + 2.0**-21 * s.abs()


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n", [50, 700])
@pytest.mark.parametrize("big", [500.0, 2000.0, 20000.0])
def test_a_feature_far_above_the_others(cuda, big, n, d, out_dtype):
    """The keys are zero there, so the score is what the other features make."""
    print(f"int8 attention outlier {big} n={n} D={d} {out_dtype}", flush=True)
    gen = torch.Generator().manual_seed(d + n)
    q = torch.randn(2, 4, 1, d, generator=gen)
    k, v = torch.randn(2, 2, 4, n, d, generator=gen)
    q[..., 3], k[..., 3] = big, 0.0
    q = q.to(torch.bfloat16).to(cuda)
    cache = filled(cuda, k.to(cuda), v.to(cuda))
    got = int8_kv_attention(q, cache, torch.tensor([n - 1], device=cuda), out_dtype=out_dtype)
    s, values, delta = scores_of(q, cache, n)
    p = s.softmax(-1)
    want = p @ values
    step, r = (2.0**-8, 15) if out_dtype == torch.bfloat16 else (2.0**-24, 23)
    bound = ((2 * delta.amax(-1, keepdim=True) + 2.0**-20) * (p @ values.abs())
             + 2.0**(5 - r) * values.abs().amax() + step * want.abs())
    assert bool(((got.double() - want).abs() <= bound).all())
