"""Capped and biased scores are formed by a polynomial where gradients are wanted and by the
exponential where they are not: how far apart the two results may be.

Either form moves a probability by at most w = 2^-12 of itself, so the two roundings to bfloat16 are
at most one step apart (2^-7 of a probability), as are those of the result: each element differs by
at most (2^-7 + 2 w) p |v| + 2^-7 |o|, and nearly all are equal."""

from __future__ import annotations

import math

import pytest
import torch

from local_ai_training.scored_attention import scored_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("cap", [5.0, 30.0, 100.0])
@pytest.mark.parametrize("std", [0.3, 1.0, 3.0])
def test_results_with_and_without_gradients(cuda, std, cap, d):
    gen = torch.Generator().manual_seed(d)
    q, k, v = ((torch.randn(2, 3, 300, d, generator=gen) * x).to(torch.bfloat16).to(cuda)
               for x in (std, std, 1.0))
    slopes = torch.tensor([0.5, 0.05, -0.02], device=cuda)
    plain = scored_attention(q, k, v, softcap=cap, slopes=slopes).double()
    wanted = scored_attention(q.clone().requires_grad_(), k, v, softcap=cap, slopes=slopes)
    at = torch.arange(300, device=cuda, dtype=torch.float64)
    s = q.double() @ k.double().transpose(2, 3).contiguous() / math.sqrt(d)
    s = cap * torch.tanh(s / cap) - slopes.double()[:, None, None] * (at[:, None] - at).abs()
    p = s.masked_fill(at[:, None] < at, -math.inf).softmax(-1)
    bound = (2.0**-7 + 2.0**-11) * (p @ v.double().abs()) + 2.0**-7 * (p @ v.double()).abs()
    apart = (wanted.detach().double() - plain).abs()
    assert bool((apart <= bound).all())
    # a result changes where a rounding falls to the other side: the forms differ by some 1e-5 of
    # a probability, a bfloat16 step is 2^-8
    assert (apart > 0).double().mean().item() < 0.1
    with torch.no_grad():
        again = scored_attention(q.clone().requires_grad_(), k, v, softcap=cap, slopes=slopes)
    assert torch.equal(again.double(), plain)
