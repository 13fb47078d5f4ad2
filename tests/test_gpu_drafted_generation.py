"""Drafted generation on the GPU: tree steps over the 8-bit and the bf16 cache, fused and through the
module forwards, and whole texts."""

from __future__ import annotations

import pytest
import torch

import draft_reference as plain
from local_ai_training.decode import fused_decode_supported
from local_ai_training.drafts import Verified, draft_tree
from local_ai_training.generate import generate
from local_ai_training.model import ModelConfig, build_seeded_model

pytestmark = pytest.mark.gpu

LETTERS = tuple(chr(48 + i) for i in range(64))
SCORES = {"attention_softcap": 20.0, "distance_bias": True}


def model_of(cuda, seed=3, mode="int8", n_layer=2, block=160, max_code=2, **kw):
    config = ModelConfig(vocab_size=64, block_size=block, n_layer=n_layer, n_head=2, n_embd=128,
                         ffn_hidden=256, matmul_mode=mode, **kw)
    return build_seeded_model(config, max_code=max_code, seed=seed).to(cuda).eval()


def tokens_of(cuda, b, s, seed=1):
    return torch.randint(0, 64, (b, s), generator=torch.Generator().manual_seed(seed + s)).to(cuda)


@pytest.mark.parametrize("scores", [{}, SCORES])
@pytest.mark.parametrize("mode,dtype", [("int8", torch.int8), ("int8", torch.bfloat16),
                                        ("int8", None), ("fp32", torch.int8), ("fp32", None)])
def test_a_chain_is_as_if_prefilled(cuda, mode, dtype, scores):
    """A chain's logits against the same tokens one by one. Over an 8-bit cache a step's own keys are
    codes, the chain's are not, and int8 rows are rounded from either: within 2^-4 of the norm."""
    print(f"chain {mode} {dtype} {bool(scores)}", flush=True)
    model = model_of(cuda, mode=mode, **scores)
    prompt, tokens = tokens_of(cuda, 2, 70), tokens_of(cuda, 2, 6, 5)
    cache, twin = (model.new_cache(2, dtype=dtype) for _ in range(2))
    model.prefill(prompt, cache)
    model.prefill(prompt, twin)
    got = model.tree_logits(tokens, draft_tree([-1, 0, 1, 2, 3, 4], cuda), cache)
    assert got.shape == (2, 6, 64) and cache.length == 70
    for i in range(6):
        want = model.decode_step(tokens[:, i:i + 1], twin).float()
        assert (got[:, i].float() - want).norm() <= 2.0**-4 * want.norm()


@pytest.mark.parametrize("scores", [{}, SCORES])
def test_fused_and_unfused_steps_agree(cuda, scores):
    """The same quantized rows up to float32 sums in another order, which move an int8 code now and
    then: within 2^-6 of the norm, as for a decode step."""
    model = model_of(cuda, **scores)
    parents = plain.random_parents(8, 1)
    prompt, tokens, tree = tokens_of(cuda, 2, 70), tokens_of(cuda, 2, 8, 5), draft_tree(parents, cuda)
    results = []
    for fused in (True, False):
        model.fused_decode = fused
        cache = model.new_cache(2, dtype=torch.int8)
        model.prefill(prompt, cache)
        assert fused_decode_supported(model, cache, 8) and not fused_decode_supported(
            model, cache, 9)
        results.append(model.tree_logits(tokens, tree, cache).float())
    assert (results[0] - results[1]).norm() <= 2.0**-6 * results[1].norm()
    model.fused_decode = True
    big = draft_tree(plain.random_parents(20, 1), cuda)  # 40 rows: not fused
    assert model.tree_logits(tokens_of(cuda, 2, 20), big, cache).shape == (2, 20, 64)


@pytest.mark.parametrize("dtype", [torch.int8, torch.bfloat16, None])
def test_committed_nodes(cuda, dtype):
    """Behind a commit the cache holds what appending those nodes one by one leaves, to the codes'
    rounding: the next step's logits within 2^-4 of the norm."""
    model = model_of(cuda)
    parents = [-1, 0, 0, 1, 2, 4]
    prompt, tokens = tokens_of(cuda, 1, 63), tokens_of(cuda, 1, 6, 5)
    cache, twin = (model.new_cache(1, dtype=dtype) for _ in range(2))
    for c in (cache, twin):
        model.prefill(prompt, c)
    model.tree_logits(tokens, draft_tree(parents, cuda), cache)
    found = Verified(torch.tensor([[0, 2, 4, -1, -1, -1]], device=cuda),
                     torch.tensor([3], device=cuda), torch.tensor([9], device=cuda))
    assert model.commit_drafts(cache, found) == ([0, 2, 4], 9)
    for i in (0, 2, 4):
        model.decode_step(tokens[:, i:i + 1], twin)
    assert cache.length == twin.length == 66 and int(cache.pos) == 66
    nine = torch.tensor([[9]], device=cuda)
    a, b = (model.decode_step(nine, c).float() for c in (cache, twin))
    assert (a - b).norm() <= 2.0**-4 * b.norm()


@pytest.mark.parametrize("shape", [(1, 1, 1), (3, 2)])
@pytest.mark.parametrize("cache_dtype", [None, torch.int8])
def test_texts(cuda, cache_dtype, shape):
    model, draft = model_of(cuda), model_of(cuda, 7, n_layer=1)
    for temperature in (0.0, 0.8):
        texts = [generate(model, LETTERS, "01234567", max_new_tokens=40, temperature=temperature,
                          top_k=30, seed=5, cache_dtype=cache_dtype, draft=draft,
                          draft_shape=shape) for _ in range(2)]
        assert texts[0] == texts[1] and len(texts[0]) == 40
    # drafted by itself, over a cache of floats: all drafts stand
    same = generate(model, LETTERS, "01234567", max_new_tokens=30, temperature=0.0, draft=model,
                    draft_shape=shape)
    assert len(same) == 30


def test_greedy_texts_in_float32_are_the_same(cuda):
    model, draft = (model_of(cuda, s, mode="fp32", max_code=None) for s in (3, 7))
    want = generate(model, LETTERS, "0123", max_new_tokens=60, temperature=0.0)
    got = generate(model, LETTERS, "0123", max_new_tokens=60, temperature=0.0, draft=draft,
                   draft_shape=(2, 2, 1))
    assert got == want


def test_texts_up_to_the_window_and_behind_it(cuda):
    model, draft = model_of(cuda, block=48), model_of(cuda, 7, n_layer=1, block=40)
    text = generate(model, LETTERS, "01234567", max_new_tokens=60, temperature=0.0,
                    cache_dtype=torch.int8, draft=draft, draft_shape=(2, 1), use_graph=True)
    assert len(text) == 60
