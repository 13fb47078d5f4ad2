"""Attention with modified scores on the CPU: the mask's plan against its definition, the torch
form against 64 bits, gradients against differences, and what is refused."""

from __future__ import annotations

import math

import pytest
import torch

from local_ai_training.scored_attention import AttentionMask, attention_mask, scored_attention
from scored_reference import layout, reference, seen_keys

KINDS = ["documents", "prefix", "documents prefix"]


def intervals(bounds, kind, s):
    at = torch.arange(s)
    return (at >= bounds[kind][..., None]) & (at < bounds[kind + 1][..., None])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("s", [1, 2, 31, 32, 33, 70])
def test_mask_is_its_definition_from_both_sides(kind, s):
    for seed in range(4):
        documents, prefix = layout(kind, 3, s, seed)
        mask = attention_mask(documents, prefix)
        seen = seen_keys(documents, prefix, 3, s)
        assert torch.equal(intervals(mask.bounds, 0, s), seen)
        assert torch.equal(intervals(mask.bounds, 2, s), seen.transpose(1, 2))
        bits = (mask.padding.long()[..., None] >> torch.arange(32)) & 1
        want = torch.zeros(3, bits.shape[1] * 32, dtype=torch.long)
        if documents is not None:
            want[:, :s] = (documents < 0).long()
        assert torch.equal(bits.reshape(3, -1), want)


def test_an_id_that_comes_back_begins_another_document():
    mask = attention_mask(torch.tensor([[5, 5, 7, 5, -1, 5]]))
    assert mask.bounds[0].tolist() == [[0, 0, 2, 3, 0, 5]]
    assert mask.bounds[1].tolist() == [[1, 2, 3, 4, 0, 6]]


@pytest.mark.parametrize("kind", ["", *KINDS])
@pytest.mark.parametrize("cap,biased", [(0.0, False), (3.0, False), (0.0, True), (3.0, True)])
def test_torch_form_against_64_bits(kind, cap, biased):
    b, h, hkv, s, d = 2, 4, 2, 21, 8
    gen = torch.Generator().manual_seed(1)
    q = torch.randn(b, h, s, d, generator=gen, requires_grad=True)
    k, v = (torch.randn(b, hkv, s, d, generator=gen, requires_grad=True) for _ in range(2))
    g = torch.randn(b, h, s, d, generator=gen)
    slopes = (0.1 * torch.rand(h, generator=gen)).requires_grad_() if biased else None
    documents, prefix = layout(kind, b, s)
    mask = attention_mask(documents, prefix) if kind else None
    out = scored_attention(q, k, v, mask=mask, softcap=cap, slopes=slopes, scale=0.7)
    leaves = [q, k, v] + ([slopes] if biased else [])
    got = [out, *torch.autograd.grad(out, leaves, g)]
    want = reference(q, k, v, g, seen_keys(documents, prefix, b, s), cap, slopes, 0.7)
    for mine, (ref, _) in zip(got, want):
        # float32: sums of at most b s s terms, each off by a few 2^-24
        assert torch.allclose(mine.double(), ref, rtol=1e-4, atol=1e-4)


def test_torch_form_against_differences():
    gen = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(1, 2, 6, 4, generator=gen, dtype=torch.float64, requires_grad=True)
               for _ in range(3))
    mask = attention_mask(torch.tensor([[0, 0, 0, -1, 1, 1]]))
    assert torch.autograd.gradcheck(
        lambda q, k, v: scored_attention(q, k, v, mask=mask, softcap=2.0,
                                         slopes=torch.tensor([0.3, 0.1])), (q, k, v),
        atol=1e-5)


def test_padding_may_hold_anything():
    documents = torch.tensor([[0, 0, -1, 1, -1]])
    mask = attention_mask(documents)
    q, k, v = (torch.randn(1, 1, 5, 4) for _ in range(3))
    clean = scored_attention(q, k, v, mask=mask)
    for t in (q, k, v):
        t[:, :, documents[0] < 0] = math.nan
    got = scored_attention(q, k, v, mask=mask)
    assert torch.equal(got, clean) and not got[:, :, 2].any()


def test_refusals():
    q = torch.randn(2, 4, 6, 8)
    k = torch.randn(2, 2, 6, 8)
    mask = attention_mask(torch.zeros(2, 6, dtype=torch.int64))
    with pytest.raises(ValueError, match="documents or prefix"):
        attention_mask()
    with pytest.raises(TypeError, match="integers"):
        attention_mask(torch.zeros(2, 6))
    with pytest.raises(TypeError, match="integers"):
        attention_mask(torch.zeros(2, 6, dtype=torch.bool))
    with pytest.raises(TypeError, match="bool"):
        attention_mask(prefix=torch.zeros(2, 6, dtype=torch.int64))
    with pytest.raises(ValueError, match="B, S"):
        attention_mask(torch.zeros(6, dtype=torch.int64))
    with pytest.raises(ValueError, match="share"):
        attention_mask(torch.zeros(2, 6, dtype=torch.int64), torch.zeros(2, 5, dtype=torch.bool))
    with pytest.raises(ValueError, match="heads"):
        scored_attention(q, torch.randn(2, 3, 6, 8), torch.randn(2, 3, 6, 8))
    with pytest.raises(ValueError, match="agree"):
        scored_attention(q, k[:, :, :5], k[:, :, :5])
    with pytest.raises(TypeError, match="dtype"):
        scored_attention(q, k.double(), k.double())
    with pytest.raises(ValueError, match="softcap"):
        scored_attention(q, k, k, softcap=-1.0)
    with pytest.raises(ValueError, match="softcap"):
        scored_attention(q, k, k, softcap=math.nan)
    with pytest.raises(ValueError, match="scale"):
        scored_attention(q, k, k, scale=0.0)
    with pytest.raises(ValueError, match="per query head"):
        scored_attention(q, k, k, slopes=torch.ones(2))
    with pytest.raises(TypeError, match="floating"):
        scored_attention(q, k, k, slopes=torch.ones(4, dtype=torch.int64))
    with pytest.raises(ValueError, match="mask"):
        scored_attention(q[:, :, :5], k[:, :, :5], k[:, :, :5], mask=mask)
    three = AttentionMask(mask.bounds[:, :1].expand(4, 3, 6), mask.padding[:1].expand(3, 1))
    with pytest.raises(ValueError, match="mask"):
        scored_attention(q, k, k, mask=three)
