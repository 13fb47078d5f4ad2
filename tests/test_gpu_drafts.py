"""Drafted trees on the GPU against 64 bits: plans, attention over the 8-bit cache, verification, and
accepted nodes into the cache.

Tolerance of the attention. Products of bfloat16 numbers (codes hold 8 bits, float32 queries are three
bfloat16 numbers to 2^-26) are exact in float32 and a score sums D of them, plus a few steps of its
scaling: it is off by at most
    delta = (D + 4) 2^-24 scale sum |q_f k_f| + 2^-21 (|raw| + |s| + cap + bias)
(the second part as for the 8-bit cache's own attention), a probability by 2 max(delta) of itself.
The sums over T tokens run over 64 at a time, then over blocks, wavefronts and splits: at most
T / 64 + 64 + 32 roundings of 2^-24, twice (numerator and denominator). bfloat16 results take
probabilities to 2^-16 and are rounded once, by 2^-8 of themselves; float32 ones by 2^-24, their
probabilities to 2^-24. Where more than 32 queries share a key head, bfloat16 results of bfloat16
queries take each probability over the cache rounded to bfloat16, by at most 2^-8 of itself: numerator
and denominator are sums of the same rounded numbers w (1 + e), |e| <= 2^-8, so a result moves by
at most sum p |e| |v - o| <= 2^-8 (sum p |v| + |o|) <= 2^-7 sum p |v|."""

from __future__ import annotations

import math

import pytest
import torch

import draft_reference as plain
from local_ai_training import drafts
from local_ai_training.drafts import (DraftTree, draft_tree, int8_kv_commit, sample_tokens,
                                      tree_attention, verify_drafts)
from local_ai_training.int8_cache import (Int8KV, int8_kv, int8_kv_append, int8_kv_attention,
                                          int8_kv_read)
from local_ai_training.ops import ratchet

pytestmark = pytest.mark.gpu


def rows(b, s, h, d, seed=0, dtype=torch.bfloat16, std=1.0):
    gen = torch.Generator().manual_seed(seed + 17 * s + d)
    return (torch.randn(b, s, h, d, generator=gen) * std).to(dtype).transpose(1, 2)


def ints(cuda, *values):
    return torch.tensor(values, dtype=torch.int64, device=cuda)


def filled(cuda, b, h, n, d, seed=0, room=0):
    cache = int8_kv(b, h, n + room or 1, d, cuda)
    if n:
        k, v = rows(b, n, h, d, seed), rows(b, n, h, d, seed + 1)
        int8_kv_append(cache, k.to(cuda), v.to(cuda), ints(cuda, 0))
    return cache


# ---------------------------------------------------------------------------
# Plans
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64, torch.int16])
@pytest.mark.parametrize("nodes", [1, 2, 63, 64, 65, 130, 256])
def test_plan(cuda, nodes, dtype):
    print(f"plan N={nodes} {dtype}", flush=True)
    parents = [plain.random_parents(nodes, seed) for seed in range(3)] + [
        [-1] + list(range(nodes - 1))]
    got = draft_tree(torch.tensor(parents, dtype=dtype).to(cuda))
    for a, b in zip(got, draft_tree(parents)):
        assert a.dtype == b.dtype and torch.equal(a.cpu(), b)


def test_nodes_with_wrong_parents_are_off(cuda):
    parents = [[-1, 0, 3, 2, 1], [-1, 0, -1, 2, 1], [0, 0, 1, 0, 3], [-1, 1, 1, 0, 3],
               [-1, 0, 2**32, 0, -2**40]]
    got = draft_tree(torch.tensor(parents).to(cuda))
    # 1, 4 | 1, 4 | none | 3, 4 (1 is its own parent, 2 its child) | 1, 3
    on = [[0, 1, 4], [0, 1, 4], [], [0, 3, 4], [0, 1, 3]]
    for r, nodes in enumerate(on):
        assert [i for i in range(5) if int(got.parents[r, i]) != -2] == nodes
        assert [i for i in range(5) if int(got.seen[r, i, 0])] == nodes
    q = torch.ones(5, 1, 5, 64, device=cuda)
    cache = filled(cuda, 5, 1, 10, 64)
    out = tree_attention(q, q, q, cache, ints(cuda, 10), got)
    for r, nodes in enumerate(on):
        assert [i for i in range(5) if out[r, 0, i].any()] == nodes
    logits = torch.zeros(5, 5, 8, device=cuda)
    found = verify_drafts(logits, torch.zeros(5, 5, dtype=torch.int64, device=cuda), got,
                          torch.zeros(5, 5, device=cuda))
    assert found.counts.tolist() == [3, 3, 0, 3, 2]


def test_plan_in_strides_and_refusals(cuda):
    wide = torch.tensor([[-1, 9, 0, 9, 0], [-1, 9, 0, 9, 1]], device=cuda)
    assert torch.equal(draft_tree(wide[:, ::2]).parents,
                       torch.tensor([[-1, 0, 0], [-1, 0, 1]], dtype=torch.int32, device=cuda))
    assert torch.equal(draft_tree([-1, 0, 0], cuda).depths, draft_tree(
        torch.tensor([-1, 0, 0], device=cuda)).depths)
    with pytest.raises(RuntimeError, match="256"):
        ratchet().draft_tree(torch.zeros(1, 257, dtype=torch.int32, device=cuda))
    torch.library.opcheck(ratchet().draft_tree, (wide.int(),))


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
def check_attention(q, k, v, cache, start, parents, lengths=None, cap=0.0, slopes=None,
                    out_dtype=None, scale=None):
    tree = draft_tree(torch.tensor(parents).to(q.device))
    got = tree_attention(q, k, v, cache, start, tree, lengths=lengths, softcap=cap or None,
                         slopes=slopes, out_dtype=out_dtype, scale=scale)
    assert got.shape == q.shape and got.dtype == (out_dtype or q.dtype)
    got_dtype, got = got.dtype, got.double().cpu()
    n, d = q.shape[2:]
    keys, values = (t.double().cpu() for t in int8_kv_read(cache))
    half = got.dtype, torch.finfo(out_dtype or q.dtype).eps / 2
    for b in range(q.shape[0]):
        s, p = int(start[b % len(start)]), parents[b % len(parents)]
        there = n if lengths is None else max(0, min(int(lengths[b]), n))
        there = 0 if s < 0 else there
        assert not got[b, :, there:].any()
        if there == 0:
            continue
        args = (t[b, :, :there].double().cpu() for t in (q, k, v))
        want, size, delta = plain.tree_attention(
            *args, keys[b, :, :s], values[b, :, :s], s, p[:there], cap,
            slopes.double().cpu() if slopes is not None else None,
            scale or 1.0 / math.sqrt(d))
        few = 2.0**-16 if (out_dtype or q.dtype) == torch.bfloat16 else 2.0**-24
        if n * q.shape[1] // k.shape[1] > 32 and q.dtype == torch.bfloat16 == got_dtype:
            few = 2.0**-7
        bound = ((2 * delta + 2 * (s / 64 + 96) * 2.0**-24 + few) * size + half[1] * want.abs())
        worst = ((got[b, :, :there] - want).abs() - bound).max().item()
        assert worst <= 0.0, (b, s, worst)


def nodes_of(cuda, b, n, heads, kv_heads, d, dtype=torch.bfloat16, seed=3):
    return (rows(b, n, heads, d, seed, dtype, 1.5).to(cuda),
            rows(b, n, kv_heads, d, seed + 1, dtype).to(cuda),
            rows(b, n, kv_heads, d, seed + 2, dtype).to(cuda))


def slopes_of(cuda, h):
    return torch.exp2(-torch.arange(1, h + 1, dtype=torch.float32, device=cuda))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("past", [0, 1, 15, 16, 63, 64, 65, 255, 300, 1000])
def test_lengths_of_the_cache(cuda, past, d):
    print(f"tree attention past={past} D={d}", flush=True)
    cache = filled(cuda, 2, 2, past, d, room=40)
    check_attention(*nodes_of(cuda, 2, 7, 2, 2, d), cache, ints(cuda, past),
                    [plain.random_parents(7, 1)])


@pytest.mark.parametrize("nodes", [1, 2, 15, 16, 17, 33, 64, 65, 130, 256])
@pytest.mark.parametrize("group", [1, 3])
def test_sizes_of_the_tree(cuda, nodes, group):
    print(f"tree attention N={nodes} G={group}", flush=True)
    cache = filled(cuda, 2, 2, 200, 64)
    check_attention(*nodes_of(cuda, 2, nodes, 2 * group, 2, 64), cache, ints(cuda, 200, 77),
                    [plain.random_parents(nodes, s) for s in range(2)])


def test_a_chain_of_all_nodes(cuda):
    cache = filled(cuda, 1, 1, 70, 128)
    check_attention(*nodes_of(cuda, 1, 256, 1, 1, 128), cache, ints(cuda, 70),
                    [[-1] + list(range(255))])


@pytest.mark.parametrize("dtype,out", [(torch.bfloat16, torch.float32),
                                       (torch.float32, torch.float32),
                                       (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_types(cuda, d, dtype, out):
    print(f"tree attention D={d} {dtype} {out}", flush=True)
    cache = filled(cuda, 2, 2, 333, d)
    for nodes, heads in ((5, 2), (20, 4)):
        check_attention(*nodes_of(cuda, 2, nodes, heads, 2, d, dtype), cache, ints(cuda, 333, 64),
                        [plain.random_parents(nodes, 2)], out_dtype=out)


@pytest.mark.parametrize("cap", [0.0, 2.0, 50.0])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_scores(cuda, cap, biased, out):
    print(f"tree attention cap={cap} bias={biased} {out}", flush=True)
    cache = filled(cuda, 2, 2, 500, 128)
    slopes = slopes_of(cuda, 4) if biased else None
    check_attention(*nodes_of(cuda, 2, 9, 4, 2, 128), cache, ints(cuda, 500, 131),
                    [plain.random_parents(9, s) for s in range(2)], cap=cap, slopes=slopes,
                    out_dtype=out, scale=0.3)
    if biased:
        check_attention(*nodes_of(cuda, 2, 9, 4, 2, 128), cache, ints(cuda, 20),
                        [plain.random_parents(9, 5)], cap=cap, slopes=-0.25 * slopes, out_dtype=out)


def test_batches_of_several_lengths(cuda):
    b = 7
    cache = filled(cuda, b, 2, 260, 64)
    start = ints(cuda, 0, 260, -1, 64, 3, 200, 130)
    lengths = ints(cuda, 12, 1, 12, 0, 400, -3, 5)
    check_attention(*nodes_of(cuda, b, 12, 4, 2, 64), cache, start,
                    [plain.random_parents(12, s) for s in range(b)], lengths=lengths)


def test_many_splits_and_tokens(cuda):
    cache = filled(cuda, 1, 1, 9000, 128)
    check_attention(*nodes_of(cuda, 1, 40, 2, 1, 128), cache, ints(cuda, 8999),
                    [plain.random_parents(40, 1)])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_token_that_takes_nearly_all(cuda, dtype):
    """One key far above the others with a small value: the result is what is left to the others."""
    cache = int8_kv(1, 1, 200, 64, cuda)
    k, v = rows(1, 190, 1, 64, 1, torch.float32), rows(1, 190, 1, 64, 2, torch.float32)
    q = rows(1, 3, 1, 64, 3, torch.float32)
    k[0, 0, 100] = 6.0 * q[0, 0, 0].sign()
    v[0, 0, 100] *= 1e-3
    int8_kv_append(cache, k.to(cuda), v.to(cuda), ints(cuda, 0))
    check_attention(q.to(cuda, dtype), *(rows(1, 3, 1, 64, s, dtype).to(cuda) for s in (4, 5)),
                    cache, ints(cuda, 190), [[-1, 0, 0]], cap=0.0)


def test_tokens_behind_the_sequence_do_not_matter(cuda):
    """Stale tokens in the last block, and blocks of NaN behind it."""
    q, k, v = nodes_of(cuda, 1, 6, 1, 1, 64)
    tree = draft_tree([plain.random_parents(6, 1)], cuda)
    full, part = filled(cuda, 1, 1, 256, 64, 5), filled(cuda, 1, 1, 256, 64, 5)
    part.keys[:, :, 2, 3:] = 99
    part.values[:, :, 2, :, 3:] = -99
    part.key_scales[:, :, 3] = math.nan
    part.value_scales[:, :, 3] = math.inf
    a, b = (tree_attention(q, k, v, c, ints(cuda, 131), tree) for c in (full, part))
    assert torch.equal(a, b) and bool(a.isfinite().all())


def test_values_that_are_not_finite(cuda):
    q, k, v = nodes_of(cuda, 1, 4, 1, 1, 64)
    tree = draft_tree([-1, 0, 0, 1], cuda)
    cache = filled(cuda, 1, 1, 100, 64)
    for name in ("key_scales", "value_scales"):
        for x in (math.nan, math.inf):
            bad = Int8KV(*(t.clone() for t in cache))
            getattr(bad, name)[:, :, 1] = x
            out = tree_attention(q, k, v, bad, ints(cuda, 65), tree)
            if name == "value_scales":
                assert not bool(out.isfinite().any())
            elif x == math.inf:  # a score of -inf has no weight, one of +inf no number
                side = (q.float() * cache.keys[0, 0, 1, 0].float()).sum(-1)
                assert torch.equal(out.isfinite().all(-1), side < 0)
                assert torch.equal(out.isnan().all(-1), side > 0)
            else:
                assert bool(out.isnan().all())
            assert bool(tree_attention(q, k, v, bad, ints(cuda, 64), tree).isfinite().all())
    for x in (math.nan, math.inf):  # node 2 and the others' ways do not meet
        kk, vv = k.clone(), v.clone()
        vv[:, :, 2, 5] = x
        kk[:, :, 3] = x
        out = tree_attention(q, kk, vv, cache, ints(cuda, 64), tree)
        assert bool(out[:, :, :2].isfinite().all())
        assert not bool(out[:, :, 2, 5].isfinite().any()) and bool(out[:, :, 3].isnan().all())


def test_starts_past_the_cache_are_nan(cuda):
    q, k, v = nodes_of(cuda, 3, 4, 1, 1, 64)
    cache = filled(cuda, 3, 1, 64, 64)
    out = tree_attention(q, k, v, cache, ints(cuda, 64, 65, 2**40), draft_tree([-1, 0, 0, 1], cuda))
    assert bool(out[0].isfinite().all()) and bool(out[1:].isnan().all())


def test_zero_blocks(cuda):
    cache = int8_kv(1, 1, 128, 64, cuda)
    zeros = torch.zeros(1, 1, 70, 64, device=cuda)
    int8_kv_append(cache, zeros, zeros, ints(cuda, 0))
    check_attention(*nodes_of(cuda, 1, 3, 1, 1, 64), cache, ints(cuda, 70), [[-1, 0, 1]],
                    out_dtype=torch.float32)


def test_strides_types_and_devices_of_operands(cuda):
    """q, k, v as parts of one projection, unaligned rows, half precision, positions in strides."""
    cache = filled(cuda, 2, 2, 90, 64)
    tree = draft_tree(plain.random_parents(5, 3), cuda)
    joint = rows(2, 5, 6, 64, 9).to(cuda).transpose(1, 2).reshape(2, 5, 384)
    q, k, v = (t.reshape(2, 5, 2, 64).transpose(1, 2) for t in joint.split(128, dim=2))
    want = tree_attention(*(t.contiguous() for t in (q, k, v)), cache, ints(cuda, 90, 40), tree)
    parts = [t.view(2, 5, 2, 64).transpose(1, 2) for t in joint.split(128, dim=2)]
    start = ints(cuda, 90, 7, 40, 7)[::2]
    assert torch.equal(tree_attention(*parts, cache, start, tree), want)
    odd = [torch.empty(2, 2, 5, 67, device=cuda, dtype=t.dtype)[..., 3:].copy_(t) for t in parts]
    assert torch.equal(tree_attention(*odd, cache, start, tree), want)
    half = tree_attention(*(t.half() for t in parts), cache, start, tree)
    single = tree_attention(*(t.half().float() for t in parts), cache, start, tree)
    assert half.dtype == torch.float16 and torch.equal(half, single.half())
    mixed = tree_attention(parts[0].float(), *parts[1:], cache, start, tree)
    assert torch.equal(mixed, tree_attention(*(t.float() for t in parts), cache, start, tree))


def test_empty_operands(cuda):
    tree = draft_tree([-1, 0], cuda)
    cache = int8_kv(2, 2, 64, 64, cuda)
    none = torch.zeros(2, 0, 2, 64, device=cuda)
    kv = torch.zeros(2, 2, 2, 64, device=cuda)
    assert tree_attention(none, kv, kv, cache, ints(cuda, 0), tree).shape == (2, 0, 2, 64)


def test_one_node_is_one_token(cuda):
    """A tree of its root alone against the attention of an appended token, up to the rounding of its
    key and value to codes."""
    q, k, v = nodes_of(cuda, 3, 1, 4, 2, 128, torch.float32)
    cache = filled(cuda, 3, 2, 150, 128, room=1)
    got = tree_attention(q, k, v, cache, ints(cuda, 150), draft_tree([-1], cuda))
    twin = Int8KV(*(t.clone() for t in cache))
    int8_kv_append(twin, k, v, ints(cuda, 150))
    kept = [t[:, :, 150:] for t in int8_kv_read(twin, 0, 151)]
    same = tree_attention(q, *kept, twin, ints(cuda, 150), draft_tree([-1], cuda))
    want = int8_kv_attention(q, twin, ints(cuda, 150))
    # 23-bit queries and float32 sums on either side: scores of size 10 to 2^-20, results of size 1
    assert (same - want).abs().max() <= 2.0**-14
    assert (got - want).abs().max() <= 0.1


def test_repeatable_on_another_stream(cuda):
    q, k, v = nodes_of(cuda, 2, 20, 4, 2, 128)
    cache = filled(cuda, 2, 2, 2000, 128)
    tree = draft_tree(plain.random_parents(20, 1), cuda)
    first = tree_attention(q, k, v, cache, ints(cuda, 2000), tree)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = tree_attention(q, k, v, cache, ints(cuda, 2000), tree)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(first, again)


def test_attention_operator(cuda):
    q, k, v = nodes_of(cuda, 1, 5, 2, 1, 64)
    cache = filled(cuda, 1, 1, 70, 64)
    tree = draft_tree(plain.random_parents(5, 1), cuda)
    args = (q, k, v, *cache, ints(cuda, 70), None, tree.depths, tree.seen, 0.125, 0.0, None,
            torch.bfloat16)
    torch.library.opcheck(ratchet().tree_attention, args)
    with pytest.raises(ValueError, match="tree"):
        ratchet().tree_attention(*args[:9], tree.depths[:, :3], *args[10:])
    with pytest.raises(ValueError, match="device"):
        ratchet().tree_attention(q, k.cpu(), *args[2:])


# ---------------------------------------------------------------------------
# Verification
# ---------------------------------------------------------------------------
def check_verification(cuda, logits, tokens, parents, uniforms, other=None, temperature=1.0,
                       top_k=None, lengths=None):
    tree = draft_tree(torch.tensor(parents).to(cuda))
    got = verify_drafts(logits.to(cuda), tokens.to(cuda), tree,
                        uniforms.to(cuda) if uniforms is not None else None,
                        draft_logits=other.to(cuda) if other is not None else None,
                        temperature=temperature, top_k=top_k,
                        lengths=lengths.to(cuda) if lengths is not None else None)
    path, counts, following = (t.cpu() for t in got)
    n = tokens.shape[1]
    for s in range(len(tokens)):
        there = n if lengths is None else min(int(lengths[s]), n)
        way, token, near = plain.verify(
            logits[s].float(), tokens[s], parents[s % len(parents)][:there],
            uniforms[s] if uniforms is not None else None,
            other[s].float() if other is not None else None, temperature, top_k)
        assert near > 1e-12, "a border case: the inputs do not decide it"
        assert path[s].tolist() == way + [-1] * (n - len(way)), s
        assert (int(counts[s]), int(following[s])) == (len(way), token), s
    return counts


def choice(b, n, vocab, seed, drafter, likely=6, dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    logits = torch.randn(b, n, vocab, generator=gen) * 2
    logits[..., :likely] += math.log(vocab) + 1.0
    other = logits + 0.7 * torch.randn(b, n, vocab, generator=gen) if drafter else None
    tokens = torch.randint(0, min(likely, vocab), (b, n), generator=gen)
    return (logits.to(dtype), tokens, torch.rand(b, n, generator=gen),
            other.to(dtype) if drafter else None)


CHOICES = [(0.0, None, False), (1.0, None, False), (1.0, None, True), (0.7, 5, False),
           (0.7, 5, True), (1.3, 1, True), (1.0, 3000, True), (0.05, None, True)]


@pytest.mark.parametrize("temperature,top_k,drafter", CHOICES)
@pytest.mark.parametrize("vocab", [1, 3, 65, 256, 1001, 8192])
def test_vocabularies(cuda, vocab, temperature, top_k, drafter):
    print(f"verify V={vocab} T={temperature} k={top_k} drafter={drafter}", flush=True)
    b, n = 8, 9
    for dtype in (torch.float32, torch.bfloat16):
        logits, tokens, uniforms, other = choice(b, n, vocab, vocab, drafter, dtype=dtype)
        parents = [plain.random_parents(n, s, 3) for s in range(b)]
        check_verification(cuda, logits, tokens, parents, uniforms, other, temperature, top_k)


@pytest.mark.parametrize("nodes", [1, 2, 31, 64, 200, 256])
@pytest.mark.parametrize("drafter", [False, True])
def test_sizes_of_verified_trees(cuda, nodes, drafter):
    print(f"verify N={nodes} drafter={drafter}", flush=True)
    logits, tokens, uniforms, other = choice(3, nodes, 300, nodes, drafter, likely=40)
    counts = check_verification(cuda, logits, tokens, [plain.random_parents(nodes, s, 8)
                                                       for s in range(3)], uniforms, other)
    assert nodes < 31 or not drafter or int(counts.max()) > 1  # (a lookup's stand by 1 in 40)


@pytest.mark.parametrize("drafter", [False, True])
def test_many_siblings(cuda, drafter):
    """One node with 40 children, among them the same tokens twice, and numbers that reject."""
    logits, tokens, uniforms, other = choice(4, 41, 500, 3, drafter, likely=30)
    check_verification(cuda, logits, tokens, [[-1] + [0] * 40], 0.9 + 0.09 * uniforms, other)


def test_a_large_vocabulary(cuda):
    logits, tokens, uniforms, other = choice(2, 3, 600_001, 1, True)
    check_verification(cuda, logits, tokens, [[-1, 0, 0]], uniforms, other)
    flat = torch.zeros(2, 3, 600_001)  # every token as likely as another
    flat[..., 7] = 0.5
    check_verification(cuda, flat, tokens, [[-1, 0, 0]], uniforms, None, top_k=1)


def test_ties_and_extreme_logits(cuda):
    """Equal logits at the k-th largest stay; zeros of either sign are equal; far apart and shifted."""
    logits = torch.zeros(4, 2, 100)
    logits[..., 50:] = -0.0
    logits[1, :, 20:40] = 1.0
    logits[2] = torch.linspace(-3e4, 3e4, 100)
    logits[3] = 1e30
    logits[3, :, ::2] = -math.inf
    tokens = torch.tensor([[0, 3], [0, 20], [0, 99], [0, 1]])
    uniforms = torch.tensor([[0.777, 0.999], [0.3, 0.01], [0.5, 0.5], [0.25, 0.001]])
    for top_k in (None, 7, 30):
        check_verification(cuda, logits, tokens, [[-1, 0]], uniforms, top_k=top_k)
    check_verification(cuda, logits, tokens, [[-1, 0]], None, temperature=0.0)


def test_numbers_at_the_ends(cuda):
    """The least and the largest random numbers."""
    logits, tokens, _, other = choice(4, 5, 700, 8, True)
    for u in (0.0, 1.0 - 2.0**-24):
        uniforms = torch.full((4, 5), u)
        check_verification(cuda, logits, tokens, [plain.random_parents(5, 2, 2)], uniforms, other)
        check_verification(cuda, logits, tokens, [plain.random_parents(5, 2, 2)], uniforms, None)


def test_the_target_as_its_own_drafter(cuda):
    """Drafts drawn from the same distribution always stand."""
    logits, tokens, uniforms, _ = choice(6, 8, 999, 5, False)
    drawn = sample_tokens(logits[:, :-1].flatten(0, 1), uniforms[:, 1:].flatten().flip(0),
                          temperature=0.6, top_k=50)
    tokens[:, 1:] = drawn.view(6, 7)
    tree = draft_tree([-1] + list(range(7)), cuda)
    got = verify_drafts(logits.to(cuda), tokens.to(cuda), tree, uniforms.to(cuda),
                        draft_logits=logits.to(cuda), temperature=0.6, top_k=50)
    assert got.counts.tolist() == [8] * 6


def test_sequences_of_several_sizes(cuda):
    logits, tokens, uniforms, other = choice(5, 12, 333, 2, True)
    parents = [plain.random_parents(12, s, 3) for s in range(5)]
    check_verification(cuda, logits, tokens, parents, uniforms, other,
                       lengths=torch.tensor([12, 1, 5, 300, 11]))
    none = verify_drafts(logits.to(cuda), tokens.to(cuda), draft_tree(parents, cuda),
                         uniforms.to(cuda), lengths=ints(cuda, 0, -5, 1, 0, 0))
    assert none.counts.tolist() == [0, 0, 1, 0, 0]
    assert none.path.tolist()[2][:2] == [0, -1] and none.path[[0, 1, 3, 4]].eq(-1).all()
    assert none.next[[0, 1, 3, 4]].eq(-1).all() and int(none.next[2]) >= 0


def test_rows_that_are_no_distribution(cuda):
    logits = torch.zeros(4, 2, 5, device=cuda)
    logits[0, 0, 3] = math.nan
    logits[1, 0, 3] = math.inf
    logits[2, 0] = -math.inf
    tokens = ints(cuda, [0, 3], [0, 3], [0, 3], [0, 3])
    tree = draft_tree([-1, 0], cuda)
    for top_k in (None, 2):
        for other in (None, torch.zeros_like(logits), logits):
            got = verify_drafts(logits, tokens, tree, torch.zeros(4, 2, device=cuda),
                                draft_logits=other, top_k=top_k)
            assert got.next[:3].tolist() == [-1] * 3 and got.counts[:3].tolist() == [1] * 3
    greedy = verify_drafts(logits, tokens, tree, temperature=0.0)  # NaN is above all numbers
    assert greedy.counts[:2].tolist() == [2, 2]


def test_unknown_tokens_do_not_stand(cuda):
    tokens = ints(cuda, [0, 7, 2], [0, -1, 2], [0, 2**40, 2**32 + 1])
    got = verify_drafts(torch.zeros(3, 3, 5, device=cuda), tokens, draft_tree([-1, 0, 0], cuda),
                        torch.zeros(3, 3, device=cuda))
    assert got.path.tolist() == [[0, 2, -1], [0, 2, -1], [0, -1, -1]]


@pytest.mark.parametrize("vocab", [250, 20000])
@pytest.mark.parametrize("drafter", [False, True])
def test_unknown_tokens_leave_the_distribution_as_it_is(cuda, drafter, vocab):
    """Trees filled up with children of no token: what stands and follows is as without them."""
    gen = torch.Generator().manual_seed(5)
    logits = torch.randn(40, 6, vocab, generator=gen)
    other = logits + torch.randn(40, 6, vocab, generator=gen) if drafter else None
    uniforms = torch.rand(40, 6, generator=gen)
    tokens = torch.randint(vocab, (40, 6), generator=gen)
    tokens[:, 1] = -1
    tokens[::2, 3] = vocab
    parents = [-1, 0, 0, 0, 1, 2]
    got = verify_drafts(logits.to(cuda), tokens.to(cuda), draft_tree(parents, cuda),
                        uniforms.to(cuda),
                        draft_logits=other.to(cuda) if drafter else None)
    want = verify_drafts(logits, tokens, draft_tree(parents), uniforms, draft_logits=other)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))


def test_logits_in_strides_and_other_types(cuda):
    logits, tokens, uniforms, other = (t.to(cuda) for t in choice(3, 6, 250, 4, True))
    tree = draft_tree(plain.random_parents(6, 1, 2), cuda)
    want = verify_drafts(logits, tokens, tree, uniforms, draft_logits=other)

    def same(*args, **kw):
        got = verify_drafts(*args, **kw)
        assert all(torch.equal(a, b) for a, b in zip(got, want))

    wide = torch.zeros(3, 13, 257, device=cuda)
    wide[:, ::2][:, :6, 5:255] = logits
    part = wide[:, ::2][:, :6, 5:255]
    same(part, tokens, tree, uniforms, draft_logits=other)
    turned = logits.transpose(1, 2).contiguous().transpose(1, 2)
    same(turned, tokens.t().contiguous().t(), tree, uniforms.t().contiguous().t(),
         draft_logits=other.transpose(0, 1).contiguous().transpose(0, 1))
    same(logits.double(), tokens, tree, uniforms, draft_logits=other)
    small = verify_drafts(logits.half(), tokens, tree, uniforms, draft_logits=other.half())
    twin = verify_drafts(logits.half().float(), tokens, tree, uniforms,
                         draft_logits=other.half().float())
    assert all(torch.equal(a, b) for a, b in zip(small, twin))


def test_sampled_tokens(cuda):
    gen = torch.Generator().manual_seed(3)
    logits, u = torch.randn(200, 777, generator=gen) * 2, torch.rand(200, generator=gen)
    for temperature, top_k in ((1.0, None), (0.5, 20), (0.0, None)):
        got = sample_tokens(logits.to(cuda), u.to(cuda), temperature=temperature, top_k=top_k)
        want = sample_tokens(logits, u, temperature=temperature, top_k=top_k)
        assert torch.equal(got.cpu(), want)


def test_logits_that_want_gradients(cuda):
    logits, tokens, uniforms, other = (t.to(cuda) for t in choice(3, 6, 250, 4, True))
    tree = draft_tree(plain.random_parents(6, 1, 2), cuda)
    want = verify_drafts(logits, tokens, tree, uniforms, draft_logits=other)
    got = verify_drafts(logits.requires_grad_(), tokens, tree, uniforms,
                        draft_logits=other.requires_grad_())
    assert all(torch.equal(a, b) and not a.requires_grad for a, b in zip(got, want))
    q, k, v = nodes_of(cuda, 1, 4, 1, 1, 64)
    cache, tree = filled(cuda, 1, 1, 70, 64), draft_tree([-1, 0, 0, 1], cuda)
    for t in (q, k, v):
        t.requires_grad_()
        with pytest.raises(RuntimeError, match="no gradient"):
            tree_attention(q, k, v, cache, ints(cuda, 70), tree)
        with torch.no_grad():
            tree_attention(q, k, v, cache, ints(cuda, 70), tree)
        t.requires_grad_(False)
    with pytest.raises(RuntimeError, match="no gradient"):
        int8_kv_commit([cache], [k.requires_grad_()], [v], ints(cuda, 0), ints(cuda, [0]),
                       ints(cuda, 1))


def test_many_sequences(cuda):
    """More rows than a launch's second and third dimensions hold."""
    gen = torch.Generator().manual_seed(1)
    logits = (torch.randn(1, 9, generator=gen) * 2).expand(70_000, 9)
    u = torch.rand(70_000, generator=gen)
    got = sample_tokens(logits.to(cuda), u.to(cuda))
    sums = logits[0].double().softmax(0).cumsum(0)
    assert (sums[None] - u.double()[:, None] * sums[-1]).abs().min() > 1e-12
    want = (sums[None] <= u.double()[:, None] * sums[-1]).sum(1)
    assert torch.equal(got.cpu(), want)


def test_verification_operator(cuda):
    logits, tokens, uniforms, other = (t.to(cuda) for t in choice(2, 4, 50, 4, True))
    tree = draft_tree([-1, 0, 0, 1], cuda)
    args = (logits, tokens, tree.parents, uniforms, None, other, 1.0, 0)
    torch.library.opcheck(ratchet().verify_drafts, args)
    for i, bad, match in ((3, None, "uniforms"), (6, -1.0, "temperature"), (7, -1, "top_k"),
                          (2, tree.parents[:, :2], "tree"), (5, other[:, :3], "shape"),
                          (1, tokens.int(), "int64")):
        with pytest.raises(ValueError, match=match):
            ratchet().verify_drafts(*args[:i], bad, *args[i + 1:])


# ---------------------------------------------------------------------------
# Accepted nodes into the cache
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("layers", [1, 3, 35])
def test_commit(cuda, layers, d, dtype):
    """Every layer's cache to the last code as appending the gathered nodes leaves it."""
    print(f"commit layers={layers} D={d} {dtype}", flush=True)
    b, h, n = 5, 2, 20
    start, counts = ints(cuda, 60, 0, 127, -1, 90), ints(cuda, 9, 20, 3, 4, 0)
    gen = torch.Generator().manual_seed(d)
    path = torch.stack([torch.randperm(n, generator=gen) for _ in range(b)]).to(cuda)
    caches = [filled(cuda, b, h, 130, d, i, room=20) for i in range(layers)]
    twins = [Int8KV(*(t.clone() for t in c)) for c in caches]
    ks = [rows(b, n, h, d, 50 + i, dtype, 1.0 + i % 3).to(cuda) for i in range(layers)]
    vs = [rows(b, n, h, d, 90 + i, dtype, 0.5 + i % 3).to(cuda) for i in range(layers)]
    int8_kv_commit(caches, ks, vs, start, path, counts)
    index = path[:, None, :, None].expand(b, h, n, d)
    for twin, k, v, cache in zip(twins, ks, vs, caches):
        int8_kv_append(twin, k.gather(2, index), v.gather(2, index), start, counts)
        assert all(torch.equal(x, y) for x, y in zip(cache, twin))


def test_commit_of_one_path(cuda):
    """One start for all, a path wider than the counts, its tail -1; nodes that are not there."""
    caches = [filled(cuda, 2, 1, 70, 64, room=64) for _ in range(2)]
    twin = Int8KV(*(t.clone() for t in caches[0]))
    k, v = (rows(2, 4, 1, 64, s).to(cuda) for s in (1, 2))
    path = ints(cuda, [0, 2, 3, -1], [0, 9, -1, -1])
    int8_kv_commit(caches, [k, k], [v, v], ints(cuda, 70), path, ints(cuda, 3, 2))
    gathered = [torch.stack([t[0][:, [0, 2, 3]], torch.cat([t[1][:, :1], 0 * t[1][:, :2]], dim=1)])
                for t in (k, v)]
    int8_kv_append(twin, *gathered, ints(cuda, 70), ints(cuda, 3, 2))
    for c in caches:
        assert all(torch.equal(x, y) for x, y in zip(c, twin))


def test_commit_past_the_cache_is_dropped(cuda):
    cache = filled(cuda, 2, 1, 64, 64)
    before = [t.clone() for t in cache]
    k = rows(2, 3, 1, 64).to(cuda)
    int8_kv_commit([cache], [k], [k], ints(cuda, 64, 2**40), ints(cuda, [0, 1, 2], [0, 1, 2]),
                   ints(cuda, 3, 3))
    assert all(torch.equal(x, y) for x, y in zip(cache, before))


def test_commit_operator(cuda):
    cache = filled(cuda, 1, 1, 64, 64, room=64)
    k = rows(1, 3, 1, 64).to(cuda)
    args = ([k], [k], *([t] for t in cache), ints(cuda, 64), ints(cuda, [0, 2, -1]), ints(cuda, 2))
    torch.library.opcheck(ratchet().int8_kv_commit, args,
                          test_utils=("test_schema", "test_faketensor"))
    with pytest.raises(ValueError, match="layer"):
        ratchet().int8_kv_commit([k, k], *args[1:])
    with pytest.raises(ValueError, match="path"):
        ratchet().int8_kv_commit(*args[:7], args[7].int(), args[8])


# ---------------------------------------------------------------------------
# Together
# ---------------------------------------------------------------------------
def test_rounds_in_a_graph(cuda):
    """A step of all four, captured once and replayed from changing inputs, against the same step run
    eagerly: attention, verification of logits made of it, the accepted nodes into the cache, the
    positions moved."""
    b, h, n, d, vocab, layers = 3, 2, 11, 64, 97, 2
    caches = [[filled(cuda, b, h, 60, d, i, room=200) for i in range(layers)] for _ in range(2)]
    head = rows(1, vocab, 1, h * d, 5, torch.float32).to(cuda)[0, 0] * 0.2
    inputs = {"q": [torch.empty(b, h, n, d, dtype=torch.bfloat16, device=cuda) for _ in range(3)],
              "parents": torch.empty(b, n, dtype=torch.int32, device=cuda),
              "tokens": torch.empty(b, n, dtype=torch.int64, device=cuda),
              "u": torch.empty(b, n, device=cuda)}
    starts = [ints(cuda, 60, 33, 60) for _ in range(2)]

    def step(side):
        tree = draft_tree(inputs["parents"])
        outs = []
        for cache in caches[side]:
            outs.append(tree_attention(*inputs["q"], cache, starts[side], tree))
        hidden = (outs[0] + outs[1]).transpose(1, 2).reshape(b * n, h * d).float()
        logits = (hidden @ head.t()).view(b, n, vocab)
        found = verify_drafts(logits, inputs["tokens"], tree, inputs["u"], temperature=0.8,
                              top_k=60)
        int8_kv_commit(caches[side], [inputs["q"][1]] * layers, [inputs["q"][2]] * layers,
                       starts[side], found.path, found.counts)
        starts[side].add_(found.counts)
        return [*outs, *found]

    def feed(turn):
        gen = torch.Generator().manual_seed(turn)
        for i, t in enumerate(inputs["q"]):
            t.copy_(rows(b, n, h, d, 10 * turn + i).to(cuda))
        inputs["parents"].copy_(torch.tensor([plain.random_parents(n, 5 * turn + s, 3)
                                              for s in range(b)]))
        inputs["tokens"].copy_(torch.randint(0, vocab, (b, n), generator=gen))
        inputs["u"].copy_(torch.rand(b, n, generator=gen) * 0.05)

    feed(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    kept = [[t.clone() for t in c] for c in caches[0]], starts[0].clone()
    with torch.cuda.stream(side):
        step(0)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(0)
    for c, old in zip(caches[0], kept[0]):
        for t, x in zip(c, old):
            t.copy_(x)
    starts[0].copy_(kept[1])
    longest = 0
    for turn in range(6):
        feed(turn)
        graph.replay()
        torch.cuda.synchronize()
        want = step(1)
        assert all(torch.equal(x, y) for x, y in zip(got, want)), turn
        for mine, other in zip(*caches):
            assert all(torch.equal(x, y) for x, y in zip(mine, other)), turn
        assert torch.equal(*starts)
        longest = max(longest, int(got[3].max()))
    assert longest > 1
