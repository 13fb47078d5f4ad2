"""The kernels of attention with modified scores against 64 bits (bounds: scored_reference.py).

Lengths: one position, the edges of the 32- and 64-row tiles and the 128-row blocks, ragged long
ones."""

from __future__ import annotations

import math

import pytest
import torch

from local_ai_training.ops import ratchet
from local_ai_training.scored_attention import (AttentionMask, _torch_mask, attention_mask,
                                                scored_attention)
from scored_reference import layout, reference, seen_keys

pytestmark = pytest.mark.gpu

KINDS = ["", "documents", "prefix", "documents prefix"]


def operands(cuda, b, h, hkv, s, d, seed=0, std=1.0):
    gen = torch.Generator().manual_seed(seed + 1000 * s + d)

    def rows(heads):
        x = torch.randn(b, s, heads, d, generator=gen) * std
        return x.to(torch.bfloat16).to(cuda).transpose(1, 2)

    return rows(h), rows(hkv), rows(hkv), rows(h)


def slopes_of(cuda, h):
    return torch.exp2(-torch.arange(1, h + 1, dtype=torch.float32, device=cuda))


def run(q, k, v, g, mask, cap, slopes, scale=None):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    if slopes is not None:
        slopes = slopes.detach().requires_grad_()
        leaves.append(slopes)
    out = scored_attention(*leaves[:3], mask=mask, softcap=cap, slopes=slopes, scale=scale)
    return [out.detach(), *torch.autograd.grad(out, leaves, g)]


def check(got, want):
    names = ("o", "dq", "dk", "dv", "dslopes")
    for name, mine, (ref, bound) in zip(names, got, want):
        assert bool(torch.isfinite(mine).all()), name
        worst = ((mine.double() - ref).abs() - bound).max().item()
        assert worst <= 0.0, (name, worst, ref.abs().max().item())


def compare(cuda, b, h, hkv, s, d, kind, cap, biased, std=1.0):
    print(f"scored attention B={b} H={h}/{hkv} S={s} D={d} {kind!r} cap={cap} {biased}",
          flush=True)
    q, k, v, g = operands(cuda, b, h, hkv, s, d, std=std)
    documents, prefix = layout(kind, b, s)
    mask = None
    if kind:
        mask = attention_mask(*(t.to(cuda) if t is not None else None
                                for t in (documents, prefix)))
    slopes = slopes_of(cuda, h) if biased else None
    got = run(q, k, v, g, mask, cap, slopes)
    check(got, reference(q, k, v, g, seen_keys(documents, prefix, b, s), cap, slopes,
                         1.0 / math.sqrt(d)))


@pytest.mark.parametrize("kind", KINDS[1:])
@pytest.mark.parametrize("s", [1, 7, 32, 33, 128, 8191, 8192, 8193, 20000])
def test_mask_equals_its_torch_form(cuda, kind, s):
    documents, prefix = layout(kind, 3, s)
    want = _torch_mask(documents, prefix)
    for dtype in (torch.int32, torch.int64):
        ids = documents.to(dtype).to(cuda) if documents is not None else None
        got = attention_mask(ids, prefix.to(cuda) if prefix is not None else None)
        for mine, ref in zip(got, want):
            assert torch.equal(mine.cpu(), ref)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("s", [1, 2, 31, 32, 33, 64, 65, 127, 128, 129, 191, 300, 517])
def test_lengths(cuda, s, d):
    compare(cuda, 2, 3, 3, s, d, "", 0.0, False)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("cap,biased", [(0.0, False), (20.0, False), (0.0, True), (20.0, True)])
@pytest.mark.parametrize("kind", KINDS)
def test_scores_and_masks(cuda, kind, cap, biased, d):
    for s in (40, 300):
        compare(cuda, 2, 4, 4, s, d, kind, cap, biased)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("h,hkv", [(6, 2), (5, 1), (8, 4)])
def test_shared_key_heads(cuda, h, hkv, d):
    compare(cuda, 2, h, hkv, 200, d, "documents prefix", 20.0, True)
    compare(cuda, 1, h, hkv, 65, d, "", 0.0, False)


@pytest.mark.parametrize("b,h", [(128, 8), (64, 16)])
def test_shared_key_heads_of_large_batches(cuda, b, h):
    """The query heads of a key head in one workgroup, and in parts of two (small batches: one)."""
    compare(cuda, b, h, 4, 130, 64, "documents", 0.0, True)


def test_scores_that_saturate_the_cap(cuda):
    compare(cuda, 1, 2, 2, 200, 128, "documents", 4.0, True, std=4.0)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("biased", [False, True])
def test_saturated_scores_with_large_values(cuda, biased, sign, d):
    """Sums of p 2^100 leave float32's range where every score is near the cap of 50 (2^72)."""
    b, h, s, scale = 2, 2, 200, 1.0 / math.sqrt(d)
    print(f"saturated D={d} {biased} sign {sign}", flush=True)
    q, k, v, g = operands(cuda, b, h, h, s, d)
    q, k = (q.abs() + 8.0), (k.abs() + 8.0) * sign
    slopes = slopes_of(cuda, h) if biased else None
    want = reference(q, k, v, g, seen_keys(None, None, b, s), 50.0, slopes, scale)
    for power in (0, 100, -60):
        with torch.no_grad():
            out = scored_attention(q, k, v * 2.0 ** power, softcap=50.0, slopes=slopes,
                                   scale=scale)
        check([out.double() * 2.0 ** -power], want)


@pytest.mark.parametrize("kind", ["", "documents prefix"])
@pytest.mark.parametrize("cap", [0.0, 20.0, 50.0])
@pytest.mark.parametrize("d", [64, 128])
def test_negative_slopes(cuda, cap, kind, d):
    """The farthest visible key counts most, and masked pairs would count more."""
    b, h, s = 2, 3, 700
    print(f"negative slopes D={d} cap={cap} {kind!r}", flush=True)
    q, k, v, g = operands(cuda, b, h, h, s, d)
    documents, prefix = layout(kind, b, s)
    mask = None
    if kind:
        mask = attention_mask(documents.to(cuda), prefix.to(cuda))
    slopes = -slopes_of(cuda, h)
    got = run(q, k, v, g, mask, cap, slopes)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = scored_attention(*leaves, mask=mask, softcap=cap, slopes=slopes)
    fixed = [out.detach(), *torch.autograd.grad(out, leaves, g)]  # slopes that do not learn
    with torch.no_grad():
        plain = scored_attention(q, k, v, mask=mask, softcap=cap, slopes=slopes)
    want = reference(q, k, v, g, seen_keys(documents, prefix, b, s), cap, slopes,
                     1.0 / math.sqrt(d))
    # Slopes of -1/2 over 700 positions take p below 2^-126, float32's smallest normal number,
    # where it is zero or a denormal: a gradient's S <= 2^10 terms p (|g| . |v| + |g| . |o|) |k|
    # with vectors of at most 128 numbers below 6 lose at most 2^-126 2^10 2 (128 36) 6 < 2^-99.
    want = [(ref, bound + 2.0 ** -99) for ref, bound in want]
    check(got, want)
    check(fixed, want)
    check([plain], want)


def test_a_long_row(cuda):
    compare(cuda, 1, 2, 1, 2500, 128, "documents prefix", 30.0, True)


def test_padding_may_hold_anything(cuda):
    q, k, v, g = operands(cuda, 2, 4, 2, 210, 128)
    documents, _ = layout("documents", 2, 210)
    documents[0, 30:60] = -1
    mask = attention_mask(documents.to(cuda))
    slopes = slopes_of(cuda, 4)
    clean = run(q, k, v, g, mask, 10.0, slopes)
    rows = (documents < 0).to(cuda)
    for t, value in ((q, math.nan), (k, math.inf), (v, -math.inf), (g, math.nan)):
        t.transpose(1, 2)[rows] = value
    got = run(q, k, v, g, mask, 10.0, slopes)
    for a, b in zip(got, clean):
        assert torch.equal(a, b)
    for t in got[:4]:
        assert not t.transpose(1, 2)[rows].any()


def test_rows_that_are_all_padding(cuda):
    q, k, v, g = operands(cuda, 2, 2, 2, 150, 64)
    documents = torch.zeros(2, 150, dtype=torch.int32)
    documents[0] = -5
    got = run(q, k, v, g, attention_mask(documents.to(cuda)), 0.0, None)
    for t in got:
        assert not t[0].any() and t[1].abs().sum() > 0


def test_one_mask_row_serves_every_sequence(cuda):
    q, k, v, g = operands(cuda, 3, 2, 2, 100, 64)
    documents, prefix = layout("documents prefix", 1, 100)
    documents, prefix = documents.to(cuda), prefix.to(cuda)
    one = run(q, k, v, g, attention_mask(documents, prefix), 0.0, None)
    many = run(q, k, v, g, attention_mask(documents.expand(3, -1), prefix.expand(3, -1)), 0.0, None)
    for a, b in zip(one, many):
        assert torch.equal(a, b)


def test_layouts_and_repeated_runs(cuda):
    q, k, v, g = operands(cuda, 2, 4, 2, 140, 128)
    slopes = slopes_of(cuda, 4)
    first = run(q, k, v, g, None, 10.0, slopes)
    again = run(*(t.contiguous() for t in (q, k, v, g)), None, 10.0, slopes)
    wide = [torch.cat([t, t], dim=-1)[..., 4:132].clone(memory_format=torch.contiguous_format)
            for t in (q, k, v, g)]
    for w, t in zip(wide, (q, k, v, g)):
        w.copy_(t)
    odd = [torch.empty(*t.shape[:3], 132, device=cuda, dtype=t.dtype)[..., 3:131].copy_(t)
           for t in wide]
    odd[3] = g.transpose(2, 3).contiguous().transpose(2, 3)
    other = run(*odd, None, 10.0, slopes)
    for a, b, c in zip(first, again, other):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_broadcast_slopes_and_gradients(cuda):
    """One slope for all heads and its gradient, every other slope of a table, a sum's gradient."""
    b, h, s, d = 2, 4, 200, 64
    q, k, v, g = operands(cuda, b, h, 2, s, d)
    seen = seen_keys(None, None, b, s)
    scale = 1.0 / math.sqrt(d)
    one = torch.full((1,), 0.125, device=cuda, requires_grad=True)
    table = slopes_of(cuda, 2 * h).requires_grad_()
    for leaf, used in ((one, one.expand(h)), (table, table[::2])):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = scored_attention(*leaves, softcap=30.0, slopes=used)
        got = [out.detach(), *torch.autograd.grad(out.sum(), [*leaves, leaf])]
        want = reference(q, k, v, torch.ones_like(g), seen, 30.0, used.detach(), scale)
        slope, bound = want[4]
        if leaf is one:
            want = (*want[:4], (slope.sum().reshape(1), bound.sum().reshape(1)))
        else:
            got[4], rest = got[4][::2], got[4][1::2]
            assert not rest.any()
        check(got, want)


def test_gradients_against_differences(cuda):
    """Along one direction, the float64 differences of the float64 formulas at the bf16 operands;
    the kernels' gradients to the bounds of their elements, summed."""
    q, k, v, g = operands(cuda, 1, 2, 1, 48, 64)
    documents, prefix = layout("documents prefix", 1, 48)
    seen = seen_keys(documents, prefix, 1, 48)
    slopes = slopes_of(cuda, 2)
    mask = attention_mask(documents.to(cuda), prefix.to(cuda))
    got = run(q, k, v, g, mask, 5.0, slopes)
    bounds = [bound for _, bound in reference(q, k, v, g, seen, 5.0, slopes, 0.125)]
    gen = torch.Generator(cuda).manual_seed(5)
    for i, x in enumerate((q, k, v, slopes)):
        way = torch.randn(x.shape, generator=gen, device=cuda, dtype=torch.float64)
        values = []
        for eps in (1e-5, -1e-5):
            moved = [t.double() for t in (q, k, v, slopes)]
            moved[i] = moved[i] + eps * way
            out = _double(moved, seen.to(cuda), 5.0, 0.125)
            values.append((out * g.double()).sum())
        slope = ((values[0] - values[1]) / 2e-5).item()
        mine = (got[1 + i].double() * way).sum().item()
        allowed = (bounds[1 + i] * way.abs()).sum().item() + 1e-6 * abs(slope) + 1e-5
        assert abs(mine - slope) <= allowed, (i, mine, slope, allowed)


def _double(tensors, seen, cap, scale):
    q, k, v, slopes = tensors
    group = q.shape[1] // k.shape[1]
    k, v = (t.repeat_interleave(group, dim=1) for t in (k, v))
    at = torch.arange(q.shape[2], device=q.device, dtype=torch.float64)
    s = cap * torch.tanh(q @ k.transpose(2, 3).contiguous() * scale / cap)
    s = s - slopes[:, None, None] * (at[:, None] - at[None, :]).abs()
    some = seen[:, None].any(-1, keepdim=True)
    p = torch.where(some, s.masked_fill(~seen[:, None], -math.inf), 0.0).softmax(-1)
    return p.masked_fill(~seen[:, None], 0.0) @ v


def test_second_derivatives_are_refused_and_batches_of_gradients_taken(cuda):
    q, k, v, g = operands(cuda, 1, 2, 2, 40, 64)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = scored_attention(*leaves, softcap=5.0)
    first = torch.autograd.grad(out.float().sum(), leaves, create_graph=True)
    for a in first:
        assert a.requires_grad
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(first[0].float().square().sum(), leaves, retain_graph=True)
    grads = torch.randn(3, *out.shape, device=cuda).bfloat16()
    got = torch.autograd.grad(out, leaves, grads, retain_graph=True, is_grads_batched=True)
    one = [torch.autograd.grad(out, leaves, x, retain_graph=True) for x in grads]
    for mine, single in zip(got, zip(*one)):
        assert torch.equal(mine, torch.stack(single))


def test_only_the_wanted_gradients(cuda):
    q, k, v, g = operands(cuda, 1, 2, 2, 40, 64)
    slopes = slopes_of(cuda, 2).requires_grad_()
    out = scored_attention(q, k, v, slopes=slopes)
    (ds,) = torch.autograd.grad(out, [slopes], g)
    want = run(q, k, v, g, None, 0.0, slopes)[-1]
    assert torch.equal(ds, want)
    with torch.no_grad():
        assert torch.equal(scored_attention(q, k, v, slopes=slopes), out)


def test_captured_and_replayed(cuda):
    """Forward and backward of several layers' shapes in one graph, replayed with other inputs
    between eager work, each replay against the eager result."""
    q, k, v, g = operands(cuda, 2, 4, 2, 150, 64)
    documents, prefix = (t.to(cuda) for t in layout("documents prefix", 2, 150))
    slopes = slopes_of(cuda, 4)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v, slopes)]

    def step():
        mask = attention_mask(documents, prefix)
        out = scored_attention(*leaves[:3], mask=mask, softcap=8.0, slopes=leaves[3])
        return [out.detach(), *torch.autograd.grad(out, leaves, g)]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(4):
        fresh = operands(cuda, 2, 4, 2, 150, 64, seed=seed)
        with torch.no_grad():
            for leaf, x in zip(leaves, fresh[:3]):
                leaf.copy_(x)
            documents.copy_(layout("documents prefix", 2, 150, seed)[0].to(cuda))
        graph.replay()
        got = [t.detach().clone() for t in captured]
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_another_stream(cuda):
    q, k, v, g = operands(cuda, 2, 2, 2, 130, 128)
    want = run(q, k, v, g, None, 5.0, None)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = run(q, k, v, g, None, 5.0, None)
    stream.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_empty_operands(cuda):
    for b, h, s in ((0, 2, 4), (2, 2, 0)):
        q = torch.zeros(b, h, s, 64, device=cuda, dtype=torch.bfloat16, requires_grad=True)
        out = scored_attention(q, q, q)
        (grad,) = torch.autograd.grad(out.sum(), [q])
        assert out.shape == grad.shape == q.shape


def test_other_types_and_head_sizes_take_the_torch_form(cuda):
    gen = torch.Generator().manual_seed(2)
    documents, prefix = layout("documents prefix", 1, 30)
    mask = attention_mask(documents.to(cuda), prefix.to(cuda))
    for dtype, d in ((torch.float32, 64), (torch.float16, 128), (torch.bfloat16, 32)):
        q, k, v = (torch.randn(1, 2, 30, d, generator=gen).to(dtype).to(cuda) for _ in range(3))
        got = scored_attention(q, k, v, mask=mask, softcap=5.0)
        want = reference(q, k, v, q, seen_keys(documents, prefix, 1, 30), 5.0, None,
                         1.0 / math.sqrt(d))[0][0]
        step = torch.finfo(dtype).eps / 2
        assert got.dtype == dtype
        assert bool(((got.double() - want).abs() <= step * want.abs() + 1e-5).all())


@pytest.mark.parametrize("cap", [1e-3, 0.5, 1e3, 1e-5, 1e6])
def test_small_and_large_caps(cuda, cap):
    """The ends of what the kernels take, and what goes to the torch form."""
    compare(cuda, 1, 2, 2, 150, 64, "documents", cap, True)


def test_empty_masks(cuda):
    for b, s in ((0, 3), (2, 0)):
        for device in ("cpu", cuda):
            mask = attention_mask(torch.zeros(b, s, dtype=torch.int64, device=device))
            assert mask.bounds.shape == (4, b, s) and mask.padding.shape == (b, -(-s // 32))


def test_the_library_refuses(cuda):
    q = torch.zeros(1, 2, 8, 64, device=cuda, dtype=torch.bfloat16)
    ops = ratchet()
    mask = attention_mask(torch.zeros(1, 8, dtype=torch.int32, device=cuda))
    with pytest.raises(RuntimeError, match="head size"):
        x = q[..., :32]
        ops.scored_attention(x, x, x, None, None, None, 0.0, 1.0, False)
    with pytest.raises(RuntimeError, match="scale"):
        ops.scored_attention(q, q, q, None, None, None, 0.0, -1.0, False)
    with pytest.raises(RuntimeError, match="softcap"):
        ops.scored_attention(q, q, q, None, None, None, -1.0, 1.0, False)
    with pytest.raises(RuntimeError, match="1e-3"):
        ops.scored_attention(q, q, q, None, None, None, 1e5, 1.0, False)
    with pytest.raises(RuntimeError, match="go together"):
        ops.scored_attention(q, q, q, mask.bounds, None, None, 0.0, 1.0, False)
    with pytest.raises(RuntimeError, match="bfloat16"):
        ops.scored_attention(q.float(), q.float(), q.float(), None, None, None, 0.0, 1.0, False)
    with pytest.raises(RuntimeError, match="multiple"):
        ops.scored_attention(q, q[:, :0], q[:, :0], None, None, None, 0.0, 1.0, False)
    with pytest.raises(RuntimeError, match="slope gradient"):
        o, lse, rest = ops.scored_attention(q, q, q, None, None, None, 0.0, 1.0, False)
        ops.scored_attention_backward(q, q, q, q, o, lse, rest, None, None, None, 0.0, 1.0, True)
    with pytest.raises(ValueError, match="device"):
        scored_attention(q, q, q, mask=AttentionMask(mask.bounds.cpu(), mask.padding.cpu()))


def test_opcheck(cuda):
    q, k, v, g = operands(cuda, 2, 4, 2, 40, 64)
    documents, prefix = (t.to(cuda) for t in layout("documents prefix", 2, 40))
    ops = ratchet()
    torch.library.opcheck(ops.attention_mask, (documents, prefix))
    mask = attention_mask(documents, prefix)
    slopes = slopes_of(cuda, 4)
    for grad in (False, True):
        torch.library.opcheck(ops.scored_attention, (q, k, v, *mask, slopes, 5.0, 0.125, grad))
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    torch.library.opcheck(ops.scored_attend, (*leaves, *mask, slopes, 5.0, 0.125))
    torch.library.opcheck(ops.scored_attend, (q, k, v, None, None, None, 0.0, 0.125))
    o, lse, rest = ops.scored_attention(q, k, v, *mask, slopes, 5.0, 0.125, True)
    for wanted in (False, True):
        torch.library.opcheck(ops.scored_attention_backward,
                              (g, q, k, v, o, lse, rest, *mask, slopes, 5.0, 0.125, wanted))
