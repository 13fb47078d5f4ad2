"""Drafted trees on the host: plans, torch forms, refusals, and that verified drafts leave the
target's distribution as it is."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import draft_reference as plain
from local_ai_training import _native as nat
from local_ai_training import drafts
from local_ai_training.drafts import (DraftTree, draft_tree, int8_kv_commit, sample_tokens,
                                      torch_tree_attention, tree_attention, verify_drafts)
from local_ai_training.int8_cache import Int8KV


@pytest.mark.parametrize("nodes", [1, 2, 5, 63, 64, 65, 200, 256])
def test_plan(nodes):
    parents = [plain.random_parents(nodes, seed) for seed in range(3)]
    tree = draft_tree(parents)
    kin = drafts._lineage(tree)
    assert kin.shape == (3, nodes, nodes) and tree.parents.tolist() == parents
    for r in range(3):
        for i in range(nodes):
            way = plain.way_of(parents[r], i)
            assert kin[r, i].nonzero().flatten().tolist() == way
            assert int(tree.depths[r, i]) == len(way) - 1


@pytest.mark.parametrize("parents", [[0], [-1, 1], [-1, 0, -1], [-1, 0, 5], [[-1, 0], [-1, 1]]])
def test_parents_on_the_host_are_checked(parents):
    with pytest.raises(ValueError, match="parent"):
        draft_tree(parents)


def test_more_trees_than_a_launch_holds():
    i64, fake = ctypes.c_int64, ctypes.c_void_p(1 << 12)  # never dereferenced
    lib = nat.load_library()
    status = lib.rk_draft_tree(fake, 0, i64(1), i64(1 << 24), i64(1), fake, fake, fake, None)
    assert status == 3 and b"too many trees" in lib.rk_last_error()
    assert lib.rk_draft_tree(fake, 0, i64(1), i64(0), i64(1), fake, fake, fake, None) == 0
    assert lib.rk_last_error() == b""


def test_plans_that_are_refused():
    with pytest.raises(ValueError, match="at most 256"):
        draft_tree([-1] + list(range(256)))
    with pytest.raises(ValueError, match="root"):
        draft_tree(torch.zeros(2, 0, dtype=torch.int64))
    with pytest.raises(ValueError, match="root"):
        draft_tree(torch.zeros(1, 1, 1, dtype=torch.int64))
    with pytest.raises(TypeError, match="integers"):
        draft_tree([-1.0, 0.0])


@pytest.mark.parametrize("cap,bias", [(0.0, False), (5.0, True)])
@pytest.mark.parametrize("start", [0, 7])
def test_attention_over_floats(start, cap, bias):
    gen = torch.Generator().manual_seed(start)

    def rand(*shape):
        return torch.randn(*shape, generator=gen, dtype=torch.float64)

    parents = [plain.random_parents(9, seed) for seed in range(2)]
    q, k, v = rand(2, 4, 9, 16), rand(2, 2, 9, 16), rand(2, 2, 9, 16)
    keys, values = rand(2, 2, 12, 16), rand(2, 2, 12, 16)
    slopes = torch.tensor([0.5, 0.25, -0.1, 0.0]).double() if bias else None
    got = torch_tree_attention(q, k, v, keys, values, start, draft_tree(parents), cap, slopes, 0.3)
    for b in range(2):
        want, size, _ = plain.tree_attention(q[b], k[b], v[b], keys[b, :, :start],
                                             values[b, :, :start], start, parents[b], cap, slopes,
                                             0.3)
        assert ((got[b] - want).abs() <= 2.0**-44 * size + 2.0**-50).all()


CHOICES = [(0.0, None, False), (1.0, None, False), (1.0, None, True), (0.7, 5, False),
           (0.7, 5, True), (1.3, 1, True), (1.0, 400, True)]


@pytest.mark.parametrize("temperature,top_k,drafter", CHOICES)
@pytest.mark.parametrize("nodes", [1, 2, 12])
def test_verification(nodes, temperature, top_k, drafter):
    gen = torch.Generator().manual_seed(nodes)
    b, vocab = 6, 40
    parents = [plain.random_parents(nodes, s, 3) for s in range(b)]
    logits = torch.randn(b, nodes, vocab, generator=gen) * 2
    other = logits + torch.randn(b, nodes, vocab, generator=gen) if drafter else None
    tokens = torch.randint(0, 6, (b, nodes), generator=gen)
    logits[..., :6] += 3.0
    uniforms = torch.rand(b, nodes, generator=gen)
    got = verify_drafts(logits, tokens, draft_tree(parents), uniforms, draft_logits=other,
                        temperature=temperature, top_k=top_k)
    for s in range(b):
        way, following, near = plain.verify(logits[s], tokens[s], parents[s], uniforms[s],
                                            other[s] if drafter else None, temperature, top_k)
        assert near > 1e-12
        assert got.path[s].tolist() == way + [-1] * (nodes - len(way))
        assert (int(got.counts[s]), int(got.next[s])) == (len(way), following)


@pytest.mark.parametrize("parents", [[-1, 0], [-1, 0, 0]])
@pytest.mark.parametrize("drafter", [False, True])
def test_tokens_are_distributed_as_the_target(drafter, parents):
    """The first new token over a fine grid of random numbers: each of its frequencies is within the
    grid's resolution of the target's probability."""
    vocab, steps = 4, 20
    p = torch.tensor([0.45, 0.3, 0.2, 0.05])
    q = torch.tensor([0.1, 0.2, 0.3, 0.4])
    n = len(parents)
    tree = draft_tree(parents)
    mass = torch.zeros(vocab, dtype=torch.float64)
    grid = (torch.arange(steps) + 0.5) / steps
    # every tuple of drafted siblings with its probability; for one draft the test's number and the
    # draw's on a grid
    kinds = torch.cartesian_prod(*[torch.arange(vocab)] * (n - 1)).view(-1, n - 1)
    numbers = torch.cartesian_prod(*[grid] * n).view(-1, n)
    if n > 2:
        numbers = torch.rand(1000, n, generator=torch.Generator().manual_seed(1))
    for row in kinds:
        weight = float(q[row].double().prod()) if drafter else float(
            torch.tensor([0.7, 0.1, 0.1, 0.1]).double()[row].prod())
        rows = len(numbers)
        tokens = torch.cat([torch.zeros(rows, 1, dtype=torch.int64), row.expand(rows, -1)], dim=1)
        logits = p.log().expand(rows, n, vocab)
        other = q.log().expand(rows, n, vocab) if drafter else None
        got = verify_drafts(logits, tokens, tree, numbers, draft_logits=other)
        second = got.path[:, 1].clamp(min=0)
        token = torch.where(got.counts > 1, tokens.gather(1, second[:, None])[:, 0], got.next)
        mass += weight * torch.bincount(token, minlength=vocab).double() / rows
    # the grid resolves each of up to 2 n borders of a unit interval to half a step; 1000 draws
    # have a deviation of at most 1 / (2 sqrt(1000)), taken five times
    bound = n / steps if n == 2 else 5 / (2 * math.sqrt(1000))
    assert (mass - p.double()).abs().max() <= bound


def test_rows_that_are_no_distribution():
    logits = torch.zeros(4, 2, 5)
    logits[0, 0, 3] = math.nan
    logits[1, 0, 3] = math.inf
    logits[2, 0] = -math.inf
    tokens = torch.tensor([[0, 3]] * 4)
    got = verify_drafts(logits, tokens, draft_tree([-1, 0]), torch.zeros(4, 2))
    assert got.next[:3].tolist() == [-1] * 3 and got.counts[:3].tolist() == [1] * 3
    assert int(got.counts[3]) == 2


def test_sequences_without_nodes_and_unknown_tokens():
    logits = torch.zeros(3, 3, 5)
    tokens = torch.tensor([[0, 7, 2], [0, -1, 2], [0, 1, 2]])
    got = verify_drafts(logits, tokens, draft_tree([-1, 0, 0]), torch.zeros(3, 3),
                        lengths=torch.tensor([3, 2, 0]))
    assert got.path.tolist() == [[0, 2, -1], [0, -1, -1], [-1, -1, -1]]
    assert got.counts.tolist() == [2, 1, 0] and got.next.tolist() == [0, 0, -1]


def test_sampled_tokens():
    logits = torch.log(torch.tensor([[0.5, 0.25, 0.25], [0.0, 1.0, 0.0]]))
    u = torch.tensor([0.6, 0.99])
    assert sample_tokens(logits, u).tolist() == [1, 1]
    assert sample_tokens(logits, temperature=0.0).tolist() == [0, 1]
    assert sample_tokens(logits, u, top_k=1).tolist() == [0, 1]


def verify_with(**kw):
    args = dict(logits=torch.zeros(2, 3, 4), tokens=torch.zeros(2, 3, dtype=torch.int64),
                tree=draft_tree([-1, 0, 0]), uniforms=torch.zeros(2, 3))
    args.update(kw)
    return verify_drafts(args.pop("logits"), args.pop("tokens"), args.pop("tree"),
                         args.pop("uniforms"), **args)


@pytest.mark.parametrize("kw,error", [
    ({"logits": torch.zeros(2, 3)}, ValueError),
    ({"logits": torch.zeros(2, 3, 0)}, ValueError),
    ({"logits": torch.zeros(2, 3, 4, dtype=torch.int64)}, ValueError),
    ({"tokens": torch.zeros(2, 3, dtype=torch.int32)}, ValueError),
    ({"tokens": torch.zeros(3, 3, dtype=torch.int64)}, ValueError),
    ({"uniforms": None}, ValueError),
    ({"uniforms": torch.zeros(2, 3, dtype=torch.float64)}, ValueError),
    ({"uniforms": torch.zeros(2, 2)}, ValueError),
    ({"draft_logits": torch.zeros(2, 3, 5)}, ValueError),
    ({"lengths": torch.zeros(3, dtype=torch.int64)}, ValueError),
    ({"temperature": -1.0}, ValueError),
    ({"temperature": math.nan}, ValueError),
    ({"temperature": 1e-9}, ValueError),
    ({"top_k": 0}, ValueError),
    ({"tree": draft_tree([-1, 0])}, ValueError),
    ({"tree": draft_tree([[-1, 0, 0]] * 3)}, ValueError),
])
def test_verifications_that_are_refused(kw, error):
    with pytest.raises(error):
        verify_with(**kw)


def cache_of(b=2, h=2, blocks=1, d=64):
    """A cache on the host: its operators refuse it, but for the checks that come first."""
    return Int8KV(torch.zeros(b, h, blocks, 64, d, dtype=torch.int8),
                  torch.zeros(b, h, blocks, d, 64, dtype=torch.int8),
                  torch.zeros(b, h, blocks), torch.zeros(b, h, blocks))


def attention_with(**kw):
    args = dict(q=torch.zeros(2, 4, 3, 64), k=torch.zeros(2, 2, 3, 64), v=torch.zeros(2, 2, 3, 64),
                cache=cache_of(), start=torch.zeros(1, dtype=torch.int64),
                tree=draft_tree([-1, 0, 0]))
    args.update(kw)
    names = ("q", "k", "v", "cache", "start", "tree")
    return tree_attention(*[args.pop(n) for n in names], **args)


@pytest.mark.parametrize("kw,error", [
    ({"q": torch.zeros(2, 3, 3, 64)}, ValueError),
    ({"q": torch.zeros(2, 4, 3, 32)}, ValueError),
    ({"q": torch.zeros(2, 4, 3, 64, dtype=torch.int8)}, TypeError),
    ({"k": torch.zeros(2, 4, 3, 64)}, ValueError),
    ({"v": torch.zeros(2, 2, 2, 64)}, ValueError),
    ({"q": torch.zeros(2, 4, 3, 64).requires_grad_()}, RuntimeError),
    ({"k": torch.zeros(2, 2, 3, 64).requires_grad_()}, RuntimeError),
    ({"slopes": torch.zeros(4).requires_grad_()}, RuntimeError),
    ({"start": torch.zeros(3, dtype=torch.int64)}, ValueError),
    ({"start": torch.zeros(1)}, ValueError),
    ({"lengths": torch.zeros(1, dtype=torch.int64)}, ValueError),
    ({"tree": draft_tree([-1, 0])}, ValueError),
    ({"tree": DraftTree(*(t[:, :2] for t in draft_tree([-1, 0, 0])))}, ValueError),
    ({"softcap": 1e-4}, ValueError),
    ({"softcap": -1.0}, ValueError),
    ({"scale": 0.0}, ValueError),
    ({"slopes": torch.zeros(2)}, ValueError),
    ({"out_dtype": torch.int32}, TypeError),
])
def test_attention_that_is_refused(kw, error):
    with pytest.raises(error):
        attention_with(**kw)


def commit_with(**kw):
    args = dict(caches=[cache_of(), cache_of()], ks=[torch.zeros(2, 2, 3, 64)] * 2,
                vs=[torch.zeros(2, 2, 3, 64)] * 2, start=torch.zeros(1, dtype=torch.int64),
                path=torch.zeros(2, 3, dtype=torch.int64),
                counts=torch.zeros(2, dtype=torch.int64))
    args.update(kw)
    return int8_kv_commit(**args)


TWICE = cache_of()


@pytest.mark.parametrize("kw,error", [
    ({"caches": []}, ValueError),
    ({"ks": [torch.zeros(2, 2, 3, 64)]}, ValueError),
    ({"caches": [TWICE, TWICE]}, ValueError),
    ({"caches": [cache_of(), cache_of(blocks=2)]}, ValueError),
    ({"vs": [torch.zeros(2, 2, 3, 64), torch.zeros(2, 2, 4, 64)]}, ValueError),
    ({"vs": [torch.zeros(2, 2, 3, 64).bfloat16()] * 2}, TypeError),
    ({"ks": [torch.zeros(2, 2, 3, 64).requires_grad_()] * 2}, RuntimeError),
    ({"path": torch.zeros(2, 3, dtype=torch.int32)}, ValueError),
    ({"path": torch.zeros(3, 3, dtype=torch.int64)}, ValueError),
    ({"counts": torch.zeros(1, dtype=torch.int64)}, ValueError),
    ({"start": torch.zeros(2)}, ValueError),
])
def test_commits_that_are_refused(kw, error):
    with pytest.raises(error):
        commit_with(**kw)
