"""Drafted texts on the GPU against undrafted ones: over a cache of floats in float32 they are the same,
over the 8-bit cache the logits of nodes in flight are near those of single steps."""

from __future__ import annotations

import pytest
import torch

from local_ai_training.drafts import draft_tree
from local_ai_training.generate import _Drafter, _TokenSampler, generate
from local_ai_training.model import ModelConfig, build_seeded_model

pytestmark = pytest.mark.gpu

LETTERS = tuple(chr(48 + i) for i in range(64))


def model_of(cuda, seed=3, block=160, n_layer=2, mode="fp32"):
    config = ModelConfig(vocab_size=64, block_size=block, n_layer=n_layer, n_head=2, n_embd=128,
                         ffn_hidden=256, matmul_mode=mode)
    code = None if mode == "fp32" else 2
    return build_seeded_model(config, max_code=code, seed=seed).to(cuda).eval()


@pytest.mark.parametrize("shape", [(1, 1, 1, 1), (3, 2)])
@pytest.mark.parametrize("temperature,top_k", [(0.0, None), (0.8, None), (0.8, 20)])
def test_a_model_that_drafts_for_itself_is_always_right(cuda, shape, temperature, top_k):
    """Every round's first way stands to its end: q is p, up to a float32 logit's rounding."""
    model = model_of(cuda)
    history = torch.arange(10, device=cuda)[None]
    caches = [model.new_cache(1) for _ in range(2)]
    for cache in caches:
        model.prefill(history, cache)
    drafter = _Drafter(model, caches[0], model, caches[1], shape,
                       _TokenSampler(temperature, top_k, 5), top_k)
    token = 11
    for turn in range(20):
        found = drafter.round(token)
        assert len(found) == len(shape) + 1, turn
        token = found[-1]
    assert caches[0].length == caches[1].length == 10 + 20 * (len(shape) + 1)


@pytest.mark.parametrize("use_graph", [False, True])
@pytest.mark.parametrize("count", [37, 40, 70])
def test_texts_up_to_the_window_and_behind_it_are_the_same(cuda, count, use_graph):
    """Windows of 48 and, the drafter's, 40: rounds, single steps, then the window anew."""
    model, draft = model_of(cuda, block=48), model_of(cuda, 7, block=40, n_layer=1)
    want = generate(model, LETTERS, "01234567", max_new_tokens=count, temperature=0.0)
    got = generate(model, LETTERS, "01234567", max_new_tokens=count, temperature=0.0, draft=draft,
                   draft_shape=(2, 1), use_graph=use_graph)
    assert got == want


@pytest.mark.parametrize("mode", ["fp32", "int8"])
def test_chains_over_the_8_bit_cache(cuda, mode):
    """A node sees itself and its ancestors as they are, a single step its own token's codes and, where
    that token raised a block's scale, the block's codes rounded once more. Codes are off by up to half
    a step, 1 / 254 of their block's largest number, so a layer's attention by some 2^-7: logits of two
    layers by less than 2^-5 of their norm in float32; int8 rows are rounded from either, within 2^-4.
    The first largest logit is another one only where two lie as near: in fewer than one step of ten."""
    model = model_of(cuda, mode=mode)
    tree, same, steps = draft_tree([-1, 0, 1, 2, 3, 4], cuda), 0, 0
    for seed in range(12):
        gen = torch.Generator().manual_seed(seed)
        prompt, tokens = (torch.randint(0, 64, (1, n), generator=gen).to(cuda) for n in (70, 6))
        cache, twin = (model.new_cache(1, dtype=torch.int8) for _ in range(2))
        model.prefill(prompt, cache)
        model.prefill(prompt, twin)
        got = model.tree_logits(tokens, tree, cache).float()[0]
        for i in range(6):
            want = model.decode_step(tokens[:, i:i + 1], twin).float()[0]
            off = (got[i] - want).norm() / want.norm()
            assert off <= (2.0**-5 if mode == "fp32" else 2.0**-4)
            same += int(got[i].argmax()) == int(want.argmax())
            steps += 1
    assert same >= 0.9 * steps
