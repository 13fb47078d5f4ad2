"""A tree's step on the host: trees and tokens that do not belong together, and steps that fail."""

from __future__ import annotations

import pytest
import torch

from local_ai_training.drafts import Verified, draft_tree
from local_ai_training.generate import generate
from local_ai_training.model import ModelConfig, build_seeded_model


def model_of(n_layer=2):
    config = ModelConfig(vocab_size=40, block_size=48, n_layer=n_layer, n_head=2, n_embd=32,
                         ffn_hidden=64)
    return build_seeded_model(config, max_code=2, seed=3).eval()


def tokens_of(b, s):
    return torch.randint(0, 40, (b, s), generator=torch.Generator().manual_seed(s))


@pytest.mark.parametrize("batch,nodes,parents", [
    (1, 1, [-1, 0, 1]), (1, 4, [-1]), (1, 3, [-1, 0]), (1, 2, [[-1, 0]] * 2), (2, 2, [[-1, 0]] * 3),
    (2, 1, [-1, 0])])
@pytest.mark.parametrize("past", [0, 5])
def test_trees_of_other_sizes_than_the_tokens_are_refused(past, batch, nodes, parents):
    model = model_of()
    cache = model.new_cache(batch)
    if past:
        model.prefill(tokens_of(batch, past), cache)
    with pytest.raises(ValueError, match="tree"):
        model.tree_logits(tokens_of(batch, nodes), draft_tree(parents), cache)
    assert cache.length == past and cache.drafted == [None, None]


def test_one_tree_for_all_or_one_for_each():
    model = model_of()
    cache, tokens = model.new_cache(2), tokens_of(2, 3)
    model.prefill(tokens_of(2, 5), cache)
    one = model.tree_logits(tokens, draft_tree([-1, 0, 0]), cache)
    each = model.tree_logits(tokens, draft_tree([[-1, 0, 0], [-1, 0, 1]]), cache)
    assert torch.equal(one[0], each[0]) and not torch.equal(one[1, 2], each[1, 2])


def test_a_step_that_fails_leaves_nothing_to_commit():
    """Half a step's keys and values beside those of an earlier one are not committed."""
    model = model_of()
    cache, tree = model.new_cache(1), draft_tree([-1, 0, 1])
    model.prefill(tokens_of(1, 5), cache)
    model.tree_logits(tokens_of(1, 3), tree, cache)

    def refuse(*args, **kw):
        raise RuntimeError("out of memory")

    last = model.blocks[1]
    forward, last.forward = last.forward, refuse
    with pytest.raises(RuntimeError, match="memory"):
        model.tree_logits((tokens_of(1, 3) + 1) % 40, tree, cache)
    last.forward = forward
    found = Verified(torch.tensor([[0, 1, -1]]), torch.tensor([2]), torch.tensor([9]))
    with pytest.raises(ValueError, match="no drafts"):
        model.commit_drafts(cache, found)
    assert cache.length == 5
    model.tree_logits(tokens_of(1, 3), tree, cache)
    assert model.commit_drafts(cache, found) == ([0, 1], 9) and cache.length == 7


@pytest.mark.parametrize("broken", ["model", "draft"])
def test_rows_that_are_no_distribution_name_both_sides(broken):
    """A residual needs both distributions: the error does not blame the model for its drafter."""
    letters = tuple(chr(48 + i) for i in range(40))
    sides = {"model": model_of(), "draft": model_of(1)}
    model, draft = sides["model"], sides["draft"]
    cached = sides[broken].tree_logits  # (a prompt's logits stay whole)
    sides[broken].tree_logits = lambda *args, **kw: cached(*args, **kw) * torch.nan
    with pytest.raises(RuntimeError, match="model's or the drafter's logits"):
        generate(model, letters, "01", max_new_tokens=6, temperature=0.9, seed=1, draft=draft,
                 draft_shape=(1, 1))
