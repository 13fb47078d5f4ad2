"""Drafted generation on the host: a tree's step over a cache of floats, its commit, and texts with a
draft model against texts without one."""

from __future__ import annotations

import pytest
import torch

import draft_reference as plain
from local_ai_training.drafts import Verified, draft_tree
from local_ai_training.generate import generate
from local_ai_training.model import ModelConfig, build_seeded_model

LETTERS = tuple(chr(48 + i) for i in range(40))


def model_of(seed=3, block=48, n_layer=2, max_code=2, **kw):
    config = ModelConfig(vocab_size=40, block_size=block, n_layer=n_layer, n_head=2, n_embd=32,
                         ffn_hidden=64, **kw)
    return build_seeded_model(config, max_code=max_code, seed=seed).eval()


def tokens_of(b, s, seed=1):
    return torch.randint(0, 40, (b, s), generator=torch.Generator().manual_seed(seed + s))


@pytest.mark.parametrize("kw", [{}, {"attention_softcap": 10.0, "distance_bias": True}])
@pytest.mark.parametrize("past", [0, 11])
def test_a_tree_step_is_the_window_of_each_way(past, kw):
    """Float32: a node's logits against the model run over the cached tokens and the node's way, to
    2^-14 of the largest (two layers' sums of 32 to 64 terms of size 1 in another order)."""
    model = model_of(**kw)
    prompt, parents = tokens_of(2, past), plain.random_parents(9, 2)
    tokens = tokens_of(2, 9, 5)
    cache = model.new_cache(2)
    if past:
        model.prefill(prompt, cache)
    got = model.tree_logits(tokens, draft_tree(parents), cache)
    assert cache.length == past and got.shape == (2, 9, 40)
    for i in range(9):
        way = torch.cat([prompt, tokens[:, plain.way_of(parents, i)]], dim=1)
        want = model(way)[0][:, -1]
        assert (got[:, i] - want).abs().max() <= 2.0**-14 * want.abs().max()


def test_committed_nodes_are_as_if_prefilled():
    model, parents = model_of(), [-1, 0, 0, 1, 2, 4]
    prompt, tokens = tokens_of(1, 7), tokens_of(1, 6, 5)
    cache, twin = model.new_cache(1), model.new_cache(1)
    model.prefill(prompt, cache)
    model.tree_logits(tokens, draft_tree(parents), cache)
    found = Verified(torch.tensor([[0, 2, 4, -1, -1, -1]]), torch.tensor([3]), torch.tensor([9]))
    assert model.commit_drafts(cache, found) == ([0, 2, 4], 9)
    model.prefill(torch.cat([prompt, tokens[:, [0, 2, 4]]], dim=1), twin)
    assert cache.length == twin.length == 10 and int(cache.pos) == 10
    a, b = (model.decode_step(torch.tensor([[9]]), c) for c in (cache, twin))
    assert (a - b).abs().max() <= 2.0**-14 * b.abs().max()
    with pytest.raises(ValueError, match="no drafts"):
        model.commit_drafts(cache, found)
    model.tree_logits(tokens, draft_tree(parents), cache)
    model.decode_step(torch.tensor([[9]]), cache)  # the cache moves on without them
    with pytest.raises(ValueError, match="no drafts"):
        model.commit_drafts(cache, found)


@pytest.mark.parametrize("shape", [(1,), (1, 1, 1, 1), (3, 2), (2, 1, 2), (4,)])
@pytest.mark.parametrize("same", [False, True])
def test_greedy_texts_are_the_same(shape, same):
    model = model_of()
    draft = model if same else model_of(7, n_layer=1)
    for prompt in ("", "0", "012345"):
        want = generate(model, LETTERS, prompt, max_new_tokens=25, temperature=0.0)
        got = generate(model, LETTERS, prompt, max_new_tokens=25, temperature=0.0, draft=draft,
                       draft_shape=shape)
        assert got == want


@pytest.mark.parametrize("count", [0, 1, 2, 41, 47, 48, 49, 60])
def test_lengths_up_to_the_window_and_behind_it(count):
    model, draft = model_of(), model_of(7, block=40, n_layer=1)
    want = generate(model, LETTERS, "01234567", max_new_tokens=count, temperature=0.0)
    assert len(want) == count
    assert generate(model, LETTERS, "01234567", max_new_tokens=count, temperature=0.0,
                    draft=draft, draft_shape=(2, 1, 1)) == want


@pytest.mark.parametrize("top_k", [None, 7])
def test_sampled_texts(top_k):
    """Seeded texts repeat, differ from seed to seed, and hold only letters within top_k."""
    model, draft = model_of(), model_of(7, n_layer=1)

    def text(seed, **kw):
        return generate(model, LETTERS, "0123", max_new_tokens=20, temperature=0.9, top_k=top_k,
                        seed=seed, draft=draft, draft_shape=(2, 2), **kw)

    assert text(1) == text(1) and len(text(1)) == 20
    assert len({text(seed) for seed in range(6)}) > 1
    if top_k:
        history = [0, 1, 2, 3]
        for letter in text(3):
            logits = model(torch.tensor([history]))[0][0, -1]
            # (within the float32 summation's reach of the k-th largest)
            assert logits[LETTERS.index(letter)] >= logits.topk(top_k).values[-1] - 2.0**-12
            history.append(LETTERS.index(letter))


def test_first_letters_are_distributed_as_without_drafts():
    """The second letter (the first that drafts touch) over 600 seeds: each frequency within five
    deviations of at most 1 / (2 sqrt(600)) of the model's probability."""
    model, draft = model_of(block=8), model_of(7, block=8, n_layer=1)
    logits = model(torch.tensor([[5]]))[0][0, -1]
    first = int(logits.argmax())
    want = (model(torch.tensor([[5, first]]))[0][0, -1] / 0.5).softmax(0)
    counts = torch.zeros(40)
    seeds = 0
    for seed in range(600):
        out = generate(model, LETTERS, LETTERS[5] + LETTERS[first], max_new_tokens=2,
                       temperature=0.5, seed=seed, draft=draft, draft_shape=(2,))
        seeds += 1
        counts[LETTERS.index(out[0])] += 1
    assert ((counts / seeds - want).abs() <= 5 / (2 * seeds**0.5)).all()


def test_refusals():
    model, draft = model_of(), model_of(7)
    other = build_seeded_model(ModelConfig(vocab_size=39, block_size=16, n_embd=32, n_head=2),
                               max_code=2, seed=1).eval()

    def text(**kw):
        return generate(model, LETTERS, "01", max_new_tokens=4, **{"draft": draft, **kw})

    for kw in ({"draft": other}, {"draft_shape": ()}, {"draft_shape": (0,)},
               {"draft_shape": (41,)}, {"draft_shape": (2,) * 8}):
        with pytest.raises(ValueError):
            text(**kw)
    cache = model.new_cache(2)
    tree = draft_tree([-1, 0])
    model.tree_logits(tokens_of(2, 2), tree, cache)
    found = Verified(torch.zeros(2, 2, dtype=torch.int64), torch.ones(2, dtype=torch.int64),
                     torch.ones(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="one sequence"):
        model.commit_drafts(cache, found)
    with pytest.raises(ValueError, match="batch"):
        model.tree_logits(tokens_of(1, 2), tree, cache)
    with pytest.raises(ValueError, match="full"):
        model.tree_logits(tokens_of(2, 49), draft_tree([-1] + list(range(48))), cache)
