"""Attention with modified scores has no forward-mode derivative: operands with a tangent are
refused, whatever else wants gradients, and never lose it without a word."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from local_ai_training.scored_attention import scored_attention

pytestmark = pytest.mark.gpu


def operands(cuda):
    gen = torch.Generator().manual_seed(0)
    rows = [torch.randn(1, 2, 40, 64, generator=gen).to(torch.bfloat16).to(cuda)
            for _ in range(3)]
    return rows + [torch.tensor([0.5, 0.25], device=cuda)]


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("grad_mode", [True, False])
def test_dual_tensors_are_refused(cuda, which, grad_mode):
    args = operands(cuda)
    with torch.set_grad_enabled(grad_mode), forward_ad.dual_level():
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises((RuntimeError, NotImplementedError), match="(?i)jvp|forward"):
            scored_attention(*args[:3], softcap=5.0, slopes=args[3])


def test_func_jvp_is_refused(cuda):
    q, k, v, slopes = operands(cuda)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: scored_attention(x, k, v, slopes=slopes), (q,),
                       (torch.ones_like(q),))


def test_a_level_without_tangents_changes_nothing(cuda):
    q, k, v, slopes = operands(cuda)
    want = scored_attention(q, k, v, slopes=slopes)
    with forward_ad.dual_level():
        assert torch.equal(scored_attention(q, k, v, slopes=slopes), want)
    with torch.no_grad():
        assert torch.equal(scored_attention(q, k, v, slopes=slopes), want)
    leaf = q.clone().requires_grad_()
    scored_attention(leaf, k, v, slopes=slopes).float().sum().backward()
    assert bool(torch.isfinite(leaf.grad).all())
