"""Verification of rows whose passes the whole device shares, or of which few logits stay, against the
plain form in 64 bits: both types, with and without a drafter, more passes than rounds, many candidates
and ties at the k-th largest."""

from __future__ import annotations

import pytest
import torch

import draft_reference as plain
from local_ai_training.drafts import draft_tree, verify_drafts

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
NEAR = 1e-12  # far above the kernels' and the plain form's error


def drafted(b, n, vocab, seed, drafter, dtype, likely, lift):
    """Logits of which the first `likely` are raised by `lift`, a drafter's beside them, drafts among
    the likely ones, random numbers."""
    gen = torch.Generator().manual_seed(seed)
    logits = torch.randn(b, n, vocab, generator=gen) * 2
    logits[..., :likely] += lift
    other = logits + 0.7 * torch.randn(b, n, vocab, generator=gen) if drafter else None
    tokens = torch.randint(0, likely, (b, n), generator=gen)
    return (logits.to(dtype), tokens, torch.rand(b, n, generator=gen),
            other.to(dtype) if drafter else None)


def wanted(logits, tokens, parents, uniforms, other, temperature, top_k):
    found = []
    for s in range(len(tokens)):
        way, token, near = plain.verify(
            logits[s].float(), tokens[s], parents, uniforms[s],
            other[s].float() if other is not None else None, temperature, top_k)
        assert near > NEAR, "a border case: the inputs do not decide it"
        found.append((way, token))
    return found


def check(cuda, logits, tokens, parents, uniforms, other=None, temperature=1.0, top_k=None):
    got = verify_drafts(logits.to(cuda), tokens.to(cuda), draft_tree(parents, cuda),
                        uniforms.to(cuda),
                        draft_logits=other.to(cuda) if other is not None else None,
                        temperature=temperature, top_k=top_k)
    n = tokens.shape[1]
    for s, (way, token) in enumerate(wanted(logits, tokens, parents, uniforms, other, temperature,
                                            top_k)):
        assert got.path[s].tolist() == way + [-1] * (n - len(way)), s
        assert (int(got.counts[s]), int(got.next[s])) == (len(way), token), s
    return got


TREES = {"chain": [-1, 0, 1, 2], "bush": [-1, 0, 0, 0, 1, 1, 2, 2]}


@pytest.mark.parametrize("vocab", [17000, 33001, 40001, 70000])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("top_k,drafter", [(None, False), (None, True), (5, False), (5, True),
                                           (600, True)])
@pytest.mark.parametrize("shape", ["chain", "bush"])
def test_large_vocabularies(cuda, shape, top_k, drafter, dtype, vocab):
    print(f"large rows V={vocab} {dtype} k={top_k} drafter={drafter} {shape}", flush=True)
    parents = TREES[shape]
    logits, tokens, uniforms, other = drafted(3, len(parents), vocab, vocab, drafter, dtype, 8, 9.0)
    check(cuda, logits, tokens, parents, uniforms, other, 0.9, top_k)


@pytest.mark.parametrize("vocab,children", [(20000, 4), (40000, 6), (70000, 9), (70000, 14)])
@pytest.mark.parametrize("top_k", [None, 9000])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_more_rejected_siblings_than_rounds(cuda, dtype, top_k, vocab, children):
    """All children of the root but the last are drafts that the target holds far less of than the
    drafter: each needs a residual of its own, more than the launches between which the device makes
    them. The last one, which the target holds more of, stands, and its children go on."""
    print(f"siblings V={vocab} {children} {dtype} k={top_k}", flush=True)
    parents = [-1] + [0] * children + [children, children]
    n = len(parents)
    logits, _, uniforms, other = drafted(2, n, vocab, children, True, dtype, 8, 6.0)
    gone = torch.arange(20, 20 + children - 1)  # drafts that the target has little of
    other[:, 0, gone] = 8.0
    logits[:, 0, gone] = 0.0
    logits[:, 0, 3], other[:, 0, 3] = 9.0, -5.0  # what is left holds the last child's
    tokens = torch.zeros(2, n, dtype=torch.int64)
    tokens[:, 1:children] = gone
    tokens[:, children] = 3
    uniforms[:, 1:children] = 1.0 - 2.0**-24
    uniforms[:, children] = 0.5
    uniforms[:, children + 1:] = 0.9
    got = check(cuda, logits, tokens, parents, uniforms, other, 1.0, top_k)
    assert got.path[:, 1].tolist() == [children] * 2


@pytest.mark.parametrize("vocab", [20000, 70000])
def test_nothing_left_between_residuals(cuda, vocab):
    """Beside rejected drafts, some that neither side holds: the residual before them stays, also where
    the walk stops for passes and goes on."""
    parents = [-1] + [0] * 11
    logits, _, uniforms, other = drafted(3, 12, vocab, 5, True, F32, 8, 6.0)
    logits[..., -2:] = -torch.inf
    other[..., -2:] = -torch.inf
    gone = torch.arange(20, 25)
    other[:, 0, gone] = 8.0
    logits[:, 0, gone] = 0.0
    logits[:, 0, 2], other[:, 0, 2] = 9.0, -5.0
    tokens = torch.zeros(3, 12, dtype=torch.int64)
    tokens[:, 1:11:2] = gone
    tokens[:, 2:12:2] = vocab - 1
    tokens[:, 11] = 2
    tokens[2, 11] = vocab - 2
    uniforms[:, 1:11] = 1.0 - 2.0**-24
    uniforms[:, 11] = 0.5
    got = check(cuda, logits, tokens, parents, uniforms, other)
    assert got.path[:, 1].tolist() == [11, 11, -1]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("drafter", [False, True])
@pytest.mark.parametrize("vocab,top_k", [(1500, 600), (1999, 1500), (5000, 513), (8192, 2500)])
def test_many_candidates(cuda, vocab, top_k, drafter, dtype):
    """More kept logits than a workgroup has threads: the k-th largest by its bits."""
    print(f"candidates V={vocab} k={top_k} {dtype} drafter={drafter}", flush=True)
    parents = plain.random_parents(6, 1, 2)
    logits, tokens, uniforms, other = drafted(4, 6, vocab, top_k, drafter, dtype, 700, 1.0)
    check(cuda, logits, tokens, parents, uniforms, other, 1.0, top_k)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("drafter", [False, True])
@pytest.mark.parametrize("vocab,ties", [(3000, 1000), (9000, 3000), (40000, 1000)])
def test_ties_at_the_kth_largest(cuda, vocab, ties, drafter, dtype):
    """Equal logits at the k-th largest all stay, in a list of candidates or over the row again."""
    print(f"ties V={vocab} {ties} {dtype} drafter={drafter}", flush=True)
    parents = [-1, 0, 0, 1]
    logits, _, uniforms, other = drafted(4, 4, vocab, ties, drafter, dtype, 20, 12.0)
    logits[..., 20:20 + ties] = 4.0
    if drafter:
        other[..., 30:30 + ties] = 4.0
    for rows in (logits, other) if drafter else (logits,):
        rows[..., 20 + ties + 10:] = rows[..., 20 + ties + 10:].clamp(max=3.5)
    tokens = torch.randint(0, 20 + ties, (4, 4), generator=torch.Generator().manual_seed(ties))
    uniforms[:, 0] = torch.tensor([0.2, 0.9, 0.99999, 0.999999])
    check(cuda, logits, tokens, parents, uniforms, other, 4.0, 40)
