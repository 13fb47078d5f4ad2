"""Sampled texts with a draft model on the host: the letters that rounds produce are distributed as the
model's own, and a model that drafts for itself is always right."""

from __future__ import annotations

import pytest
import torch

from local_ai_training.generate import _Drafter, _TokenSampler, generate
from local_ai_training.model import ModelConfig, build_seeded_model

LETTERS = tuple("abcdef")


@pytest.fixture(autouse=True)
def one_thread():
    """Rows of 32 numbers: threads only wait for each other."""
    threads = torch.get_num_threads()
    torch.set_num_threads(1)
    yield
    torch.set_num_threads(threads)


def model_of(seed, **kw):
    config = ModelConfig(**{"vocab_size": 6, "block_size": 12, "n_layer": 1, "n_head": 2,
                            "n_embd": 32, "ffn_hidden": 64, **kw})
    return build_seeded_model(config, max_code=2, seed=seed).eval()


@torch.no_grad()
def next_letters(model, history, temperature, top_k):
    row = model(torch.tensor([history]))[0][0, -1].double() / temperature
    if top_k:
        row = row.masked_fill(row < row.topk(top_k).values[-1], -torch.inf)
    return row.softmax(0)


def chances(model, source, history, temperature, top_k):
    """Of the second and third letter behind `history`: the first one `model`'s, those `source`'s."""
    second, third = torch.zeros(6).double(), torch.zeros(6).double()
    for a, pa in enumerate(next_letters(model, history, temperature, top_k).tolist()):
        row = next_letters(source, history + [a], temperature, top_k)
        second += pa * row
        for b, pb in enumerate(row.tolist()):
            third += pa * pb * next_letters(source, history + [a, b], temperature, top_k)
    return second, third


@pytest.mark.parametrize("shape,top_k", [((1, 1), None), ((2, 2), 3)])
def test_letters_behind_the_first_are_distributed_as_without_drafts(shape, top_k):
    """The first letter is drawn before any draft; rounds make the second and the third. Each letter's
    frequency over the seeds lies within five deviations of the model's probability, and the
    drafter's own probabilities do not."""
    model, draft = model_of(3), model_of(7)
    seeds, temperature = 700, 0.3
    counts = torch.zeros(2, 6).double()
    for seed in range(seeds):
        text = generate(model, LETTERS, "c", max_new_tokens=3, temperature=temperature, top_k=top_k,
                        seed=seed, draft=draft, draft_shape=shape)
        for place in (0, 1):
            counts[place, LETTERS.index(text[1 + place])] += 1
    own, other = (chances(model, source, [2], temperature, top_k) for source in (model, draft))
    for place in (0, 1):
        want = own[place]
        bound = 5 * (want * (1 - want) / seeds).sqrt() + 1e-9
        assert ((counts[place] / seeds - want).abs() <= bound).all(), place
        assert ((other[place] - want).abs() > bound).any(), place


@pytest.mark.parametrize("shape", [(1, 1, 1), (3, 2), (2,)])
@pytest.mark.parametrize("temperature,top_k", [(0.0, None), (0.8, None), (0.8, 4)])
def test_a_model_that_drafts_for_itself_is_always_right(shape, temperature, top_k):
    """Every round's first way stands to its end: q is p, up to a float32 logit's rounding."""
    model = model_of(3, block_size=40, n_layer=2)
    history = torch.tensor([[1, 2, 3]])
    caches = [model.new_cache(1) for _ in range(2)]
    for cache in caches:
        model.prefill(history, cache)
    drafter = _Drafter(model, caches[0], model, caches[1], shape,
                       _TokenSampler(temperature, top_k, 5), top_k)
    token, length = 4, 3
    while drafter.fits():
        found = drafter.round(token)
        assert len(found) == len(shape) + 1
        token, length = found[-1], length + len(found)
        assert caches[0].length == caches[1].length == length
    assert length + len(shape) >= 40
