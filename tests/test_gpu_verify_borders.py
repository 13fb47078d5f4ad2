"""Verification close to its borders: decisions that differ by a few 2^-44 are made as in 64 bits, and a
residual that is rounding alone counts as nothing."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from local_ai_training.drafts import draft_tree, sample_tokens, verify_drafts

pytestmark = pytest.mark.gpu


def borders(count):
    """Logits -d of a second token beside a first one's zero, and float32 numbers u that its
    probability p = 1 / (1 + e^d) passes or misses by 2^-44 to 2^-41 of itself. The exponents
    d log2(e) lie near the middle between 32nds, where a series around the nearest is longest. (In
    float64 p is off by a few 2^-53.)"""
    gen = np.random.default_rng(1)
    kept = []
    while sum(len(d) for d, _ in kept) < count:
        d = gen.uniform(0.5, 3.0, 4_000_000).astype(np.float32)
        p = 1.0 / (1.0 + np.exp(d.astype(np.float64)))
        u = p.astype(np.float32)
        off = np.abs(p - u.astype(np.float64)) / p
        steps = d.astype(np.float64) * (32.0 / np.log(2.0))
        middle = np.abs(steps - np.rint(steps)) > 0.45
        chosen = (off > 2.0**-44) & (off < 2.0**-41) & middle
        kept.append((d[chosen], u[chosen]))
    d, u = (np.concatenate(x)[:count] for x in zip(*kept))
    return torch.from_numpy(d), torch.from_numpy(u)


@pytest.mark.parametrize("vocab", [2, 20000])
def test_decisions_near_a_border(cuda, vocab):
    """A drafted token of probability p stands if u < p. An exponential off by e of itself moves p by
    e (1 - p) of itself: the nearest border of 2^-44 takes one to a few 2^-49."""
    d, u = borders(60)
    p = 1.0 / (1.0 + torch.exp(d.double()))
    assert len(d) == 60 and bool((p > u.double()).any()) and bool((p < u.double()).any())
    logits = torch.full((60, 2, vocab), -torch.inf)
    logits[:, :, 0], logits[:, :, 1] = 0.0, -d[:, None]
    tokens = torch.tensor([[0, 1]]).expand(60, 2).contiguous()
    uniforms = torch.stack([torch.full_like(u, 0.5), u], dim=1)
    got = verify_drafts(logits.to(cuda), tokens.to(cuda), draft_tree([-1, 0], cuda),
                        uniforms.to(cuda))
    assert torch.equal(got.counts.cpu() == 2, p > u.double())


def test_draws_near_a_border(cuda):
    """The first of two tokens is drawn if its share of their sum passes u: 1 - p against 1 - u, both
    exact where u is a multiple of 2^-24."""
    d, u = borders(400)
    whole = (u.double() * 2**24 == (u.double() * 2**24).round())
    d, u = d[whole], u[whole]
    assert len(d) > 20
    p = 1.0 / (1.0 + torch.exp(d.double()))
    first = (1.0 - u.double()).float()  # exact
    logits = torch.stack([torch.zeros_like(d), -d], dim=1)
    got = sample_tokens(logits.to(cuda), first.to(cuda))
    # the first token's border 1 - p lies above `first` where p < u
    assert torch.equal(got.cpu() == 0, p < u.double())


@pytest.mark.parametrize("vocab,top_k", [(300, 5), (300, None), (1200, 600), (40000, 5),
                                         (70000, 5), (70000, None)])
@pytest.mark.parametrize("shift", [0.0, 4.0])
def test_drafts_that_neither_side_holds(cuda, vocab, top_k, shift):
    """The drafter's logits are the target's plus a constant (multiples of 2^-8: exact), and drafted
    tokens have no probability on either side: nothing is left of p - q, so p stays, whatever the
    number of such drafts, and the draw is the target's own."""
    print(f"nothing left V={vocab} k={top_k} shift={shift}", flush=True)
    gen = torch.Generator().manual_seed(vocab)
    logits = torch.round(torch.randn(4, 4, vocab, generator=gen) * 512) / 256
    logits[..., -3:] = -torch.inf if top_k is None else -20.0
    logits[..., :40] += 6.0
    tokens = torch.tensor([[0, vocab - 1, vocab - 2, vocab - 3]]).expand(4, 4).contiguous()
    uniforms = torch.rand(4, 4, generator=gen)
    got = verify_drafts(logits.to(cuda), tokens.to(cuda), draft_tree([-1, 0, 0, 0], cuda),
                        uniforms.to(cuda), draft_logits=(logits + shift).to(cuda), top_k=top_k)
    want = sample_tokens(logits[:, 0], uniforms[:, 0], top_k=top_k)
    assert got.counts.tolist() == [1] * 4 and torch.equal(got.next.cpu(), want)
