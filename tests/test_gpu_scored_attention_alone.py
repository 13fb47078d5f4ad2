"""A token that sees only itself: its output is its value and no gradient reaches its query and key
(a softmax of one score is constant).

Tolerance. o is v, a bfloat16 number, so delta = g . o and the product g . v are the same sum of D
products in float32 in two orders. With g = v the products are positive, the partial sums grow evenly,
and each sum is off by at most D / 2 roundings of 2^-24 of the whole: their difference, the gradient of the score,
by D 2^-24 sum v^2, and dq (dk) by that times scale |k| (|q|), within the roundings of p and of the
result (1 + 2^-7)."""

from __future__ import annotations

import math

import pytest
import torch

from local_ai_training.scored_attention import attention_mask, scored_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("s", [1, 70, 300])
@pytest.mark.parametrize("cap,biased", [(0.0, False), (20.0, False), (0.0, True), (20.0, True)])
def test_no_gradient_reaches_its_query_and_key(cuda, cap, biased, s, d):
    gen = torch.Generator().manual_seed(s + d)
    q, k, v = (torch.randn(2, 3, s, d, generator=gen).to(torch.bfloat16).to(cuda).requires_grad_()
               for _ in range(3))
    slopes = torch.tensor([0.5, 0.1, -0.1], device=cuda, requires_grad=True) if biased else None
    mask = attention_mask(torch.arange(s, device=cuda).expand(2, s)) if s > 1 else None
    out = scored_attention(q, k, v, mask=mask, softcap=cap, slopes=slopes)
    assert torch.equal(out, v)
    leaves = [q, k, v] + ([slopes] if biased else [])
    dq, dk, dv, *rest = torch.autograd.grad(out, leaves, v.detach())
    off = (1.0 + 2.0**-7) * d * 2.0**-24 * v.double().square().sum(-1, keepdim=True) / math.sqrt(d)
    for name, got, other in (("dq", dq, k), ("dk", dk, q)):
        worst = (got.double().abs() / (off * other.double().abs())).nan_to_num().max().item()
        print(f"{name}: largest error / bound {worst:.3f}", flush=True)
        assert worst <= 1.0
    assert torch.equal(dv, v)
    if biased:
        assert not rest[0].any()  # no distance, whatever the products
