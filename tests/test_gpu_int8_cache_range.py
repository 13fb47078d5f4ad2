"""Attention over the 8-bit cache where numbers of very different size meet, against 64 bits over
the values the codes stand for: a feature far above a query's others, a token that takes nearly all of
the attention and whose value is zero.

Tolerance. A query is a fixed-point number of 127 256^2 steps, off by at most half a step, 2^-23.98
of its row's largest feature; its digits' integer sums are exact, and joining them in float32 takes
2^-9 of a step times the codes' sum and 2^-24 of the score. So a score is off by at most
    delta = 2^-23 scale max|q| sum|k| + 2^-21 |s|
(twice the half step, and the roundings of scales, exponentials' arguments and sums), a probability
by 2 max(delta) of itself and 2^-20 for exponentials and sums. Probabilities enter their products as
sums of bfloat16 numbers, three for float32 results and two for bfloat16 ones (one in chunks of 32
tokens and more): off by 2^-24, 2^-16 (2^-8) of themselves, whatever the others are. Results are
rounded once."""

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


def check(q, cache, n, out_dtype):
    """The last q.shape[2] of n positions."""
    new, d = q.shape[2:]
    got = int8_kv_attention(q, cache, torch.tensor([n - new], device=q.device),
                            out_dtype=out_dtype)
    keys, values = (t.double() for t in int8_kv_read(cache, 0, n))
    scale = 1.0 / math.sqrt(d)
    x = q.double()
    s = x @ keys.transpose(2, 3).contiguous() * scale
    size = scale * x.abs().amax(-1, keepdim=True) * keys.abs().sum(-1)[:, :, None]
    unseen = torch.ones_like(s, dtype=torch.bool).triu(n - new + 1)
    delta = (2.0**-23 * size + 2.0**-21 * s.abs()).masked_fill(unseen, 0.0)
    p = s.masked_fill(unseen, -math.inf).softmax(-1)
    want = p @ values
    step, rounded = 2.0**-24, 2.0**-24
    if out_dtype == torch.bfloat16:
        step, rounded = 2.0**-8, 2.0**-8 if new >= 32 and d <= 128 else 2.0**-16
    bound = ((2 * delta.amax(-1, keepdim=True) + 2.0**-20 + rounded) * (p @ values.abs())
             + step * want.abs())
    worst = ((got.double() - want).abs() / bound).max().item()
    print(f"  largest error / bound {worst:.3f}", flush=True)
    assert worst <= 1.0


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
    check(q, cache, n, out_dtype)


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 7, 40])
@pytest.mark.parametrize("n", [50, 700, 5000])
@pytest.mark.parametrize("rest", [0.1, 1e-3, 1e-6])
def test_a_token_that_takes_nearly_all(cuda, rest, n, new, d, out_dtype):
    """The first token's key lies along a feature that the queries share and the other keys do
    not have; it leaves about `rest` to the others, whose values are the result."""
    print(f"int8 attention sink rest={rest} n={n} new={new} D={d} {out_dtype}", flush=True)
    gen = torch.Generator().manual_seed(d + n + new)
    q = torch.randn(2, 3, new, d, generator=gen)
    k, v = torch.randn(2, 2, 3, n, d, generator=gen)
    q[..., 0], k[..., 0] = 12.0, 0.0
    k[:, :, 0], v[:, :, 0] = 0.0, 0.0
    k[:, :, 0, 0] = (math.log(n) + 0.5 - math.log(rest)) * math.sqrt(d) / 12.0
    cache = filled(cuda, k.to(cuda), v.to(cuda))
    check(q.to(torch.bfloat16).to(cuda), cache, n, out_dtype)
