"""The 8-bit key/value cache against plain forms: its codes to the last one (float32 quotients are
IEEE on either side), its attention against 64 bits over the values the codes stand for.

Tolerance of the attention. Queries and probabilities are fixed-point numbers of r = 23 bits for
float32 results and 15 for bfloat16 ones (127 256^2 and 127 256 steps, so half a step is below
2^-(r + 1) of the largest). A query is off by that of its row's largest feature, the float32
combination of its digits' sums by 2^-22 of |q| . |k| <= max|q| sum|k|, a capped score by 2^-21 of
the cap and the scaled, biased score by 2^-21 of itself and of the bias: a score is off by at most
    delta = (2^-21 + 2^-(r + 1)) scale max|q| sum|k| + 2^-21 (|s| + cap + slope |i - j|),
a probability by 2 max(delta) of itself, plus 2^-20 for the exponentials and sums. The fixed-point
probabilities are off by 2^-(r + 1) of their block's largest each, over 64 tokens 2^(5 - r) of the
values' largest. bfloat16 results are rounded once, by 2^-8 of themselves. Chunks of 32 bfloat16
tokens and more with bfloat16 results take bfloat16 products: each probability times its block's
value scale is rounded to bfloat16, by at most 2^-8 of itself, which moves a result by at most
2^-8 of the sum of p |v| more (the codes and the queries enter as they are)."""

from __future__ import annotations

import math

import pytest
import torch

from local_ai_training.int8_cache import (BLOCK, Int8KV, int8_kv, int8_kv_append,
                                          int8_kv_attention, int8_kv_read)
from local_ai_training.ops import ratchet

pytestmark = pytest.mark.gpu


class PlainCache:
    """The quantization rule on the CPU, a sequence and block at a time."""

    def __init__(self, b, h, max_len, d):
        self.blocks = -(-max_len // BLOCK)
        self.codes = torch.zeros(2, b, h, self.blocks * BLOCK, d)
        self.scales = torch.zeros(2, b, h, self.blocks)

    def append(self, k, v, start, lengths=None):
        for i, x in enumerate((k, v)):
            x = x.float().cpu()
            for b in range(x.shape[0]):
                p = int(start[b % len(start)])
                n = x.shape[2] if lengths is None else min(int(lengths[b]), x.shape[2])
                if p >= 0:
                    self._append(self.codes[i, b], self.scales[i, b], x[b], p,
                                 min(n, self.blocks * BLOCK - p))

    def _append(self, codes, scales, x, p, n):
        for low in range(p // BLOCK * BLOCK, p + n, BLOCK):
            first, last = max(low, p), min(low + BLOCK, p + n)
            if first >= last:
                continue
            part, j = x[:, first - p:last - p], low // BLOCK
            s = part.abs().amax((1, 2)) / torch.tensor(127.0)
            if first > low:
                old = scales[:, j]
                s = torch.maximum(s, old)
                again = (codes[:, low:first] * (old / s.where(s > 0, 1.0))[:, None, None]).round()
                codes[:, low:first] = again
            scales[:, j] = s
            codes[:, first:last] = (part / s.where(s > 0, 1.0)[:, None, None]).round()

    def values(self):
        return self.codes * self.scales.repeat_interleave(BLOCK, dim=3)[..., None]


def rows(b, s, h, d, seed=0, dtype=torch.bfloat16, std=1.0):
    gen = torch.Generator().manual_seed(seed + 17 * s + d)
    return (torch.randn(b, s, h, d, generator=gen) * std).to(dtype).transpose(1, 2)


def same_values(cache, plain, n):
    for got, want in zip(int8_kv_read(cache, 0, n), plain.values()):
        assert torch.equal(got.cpu(), want[:, :, :n])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_appended_in_parts(cuda, d, dtype):
    """Prompts, single tokens that raise a block's scale or do not, chunks that end and begin
    inside blocks."""
    b, h, max_len = 2, 3, 320
    cache, plain = int8_kv(b, h, max_len, d, cuda), PlainCache(b, h, max_len, d)
    at = 0
    for step, n in enumerate((1, 1, 61, 1, 1, 63, 64, 2, 100, 1, 25)):
        print(f"append D={d} {dtype} at {at} n={n}", flush=True)
        k, v = (rows(b, n, h, d, 10 * step + i, dtype, 0.2 + 0.3 * step) for i in range(2))
        start = torch.tensor([at])
        int8_kv_append(cache, k.to(cuda), v.to(cuda), start.to(cuda))
        plain.append(k, v, start)
        at += n
        same_values(cache, plain, at)
    assert at == cache.capacity


def test_an_old_block_is_started_anew(cuda):
    cache, plain = int8_kv(1, 2, 128, 64, cuda), PlainCache(1, 2, 128, 64)
    for start, n, std in ((0, 128, 50.0), (64, 3, 0.01), (67, 2, 0.02)):
        k, v = rows(1, n, 2, 64, start, std=std), rows(1, n, 2, 64, start + 1, std=std)
        int8_kv_append(cache, k.to(cuda), v.to(cuda), torch.tensor([start], device=cuda))
        plain.append(k, v, [start])
    same_values(cache, plain, 69)


def test_sequences_of_several_lengths(cuda):
    b, h, d, max_len = 5, 2, 128, 256
    cache, plain = int8_kv(b, h, max_len, d, cuda), PlainCache(b, h, max_len, d)
    for n, start, lengths in ((90, [0, 0, 0, 0, 0], [90, 1, 64, 0, 37]),
                              (1, [90, 1, 64, -1, 37], None),
                              (70, [91, 2, 65, 0, 250], [70, 200, 5, -3, 70])):
        k, v = rows(b, n, h, d, n), rows(b, n, h, d, n + 1, std=2.0)
        t = torch.tensor(start)
        ln = torch.tensor(lengths) if lengths else None
        int8_kv_append(cache, k.to(cuda), v.to(cuda), t.to(cuda),
                       ln.to(cuda) if lengths else None)
        plain.append(k, v, start, lengths)
    same_values(cache, plain, max_len)


def test_positions_past_the_cache_are_dropped(cuda):
    cache = int8_kv(2, 1, 64, 64, cuda)
    before = [t.clone() for t in cache]
    x = rows(2, 3, 1, 64).to(cuda)
    int8_kv_append(cache, x, x, torch.tensor([64, 2**40], device=cuda))
    for a, b in zip(cache, before):
        assert torch.equal(a, b)


def test_zeros_and_values_that_are_not_finite(cuda):
    cache = int8_kv(1, 3, 64, 64, cuda)
    x = torch.zeros(1, 3, 2, 64, device=cuda)
    x[0, 1, 0, 5] = math.nan
    x[0, 2, 1, 7] = math.inf
    int8_kv_append(cache, x, x, torch.zeros(1, dtype=torch.int64, device=cuda))
    for t in int8_kv_read(cache, 0, 2):
        assert not t[0, 0].any() and bool(t[0, 1:].isnan().any(-1).all())
    q = torch.ones(1, 3, 1, 64, device=cuda)
    out = int8_kv_attention(q, cache, torch.tensor([1], device=cuda))
    assert not out[0, 0].any() and bool(out[0, 1:].isnan().all())


def check_attention(q, cache, start, lengths=None, cap=0.0, slopes=None, out_dtype=None):
    scale = 1.0 / math.sqrt(q.shape[3])
    got = int8_kv_attention(q, cache, start, lengths=lengths, softcap=cap, slopes=slopes,
                            out_dtype=out_dtype)
    assert got.dtype == (out_dtype or q.dtype) and got.shape == q.shape
    keys, values = (t.double() for t in int8_kv_read(cache))
    group = q.shape[1] // keys.shape[1]
    keys, values = (t.repeat_interleave(group, dim=1) for t in (keys, values))
    step = torch.finfo(got.dtype).eps / 2
    r = 23 if got.dtype == torch.float32 else 15
    rounded = q.dtype == got.dtype == torch.bfloat16 and q.shape[2] >= 32 and q.shape[3] <= 128
    for b in range(q.shape[0]):
        p0 = int(start[b % len(start)])
        n = q.shape[2] if lengths is None else max(0, min(int(lengths[b]), q.shape[2]))
        n = 0 if p0 < 0 else n
        assert not got[b, :, n:].any()
        if n == 0:
            continue
        x = q[b, :, :n].double().contiguous()
        total = p0 + n
        k, v = keys[b, :, :total].contiguous(), values[b, :, :total].contiguous()
        at = p0 + torch.arange(n, device=q.device, dtype=torch.float64)
        dist = at[:, None] - torch.arange(total, device=q.device, dtype=torch.float64)
        s = x @ k.transpose(1, 2).contiguous() * scale
        if cap:
            s = cap * torch.tanh(s / cap)
        bias = slopes.double()[:, None, None] * dist.abs() if slopes is not None else 0.0
        s = s - bias
        products = scale * x.abs().amax(-1, keepdim=True) * k.abs().sum(-1)[:, None]
        size = abs(bias)  # (slopes may be negative)
        delta = 2.0**-21 * (products + s.abs() + cap + size) + 2.0**-(r + 1) * products
        unseen = dist < 0
        p = s.masked_fill(unseen, -math.inf).softmax(-1)
        want = p @ v
        bound = ((2 * delta.masked_fill(unseen, 0.0).amax(-1, keepdim=True) + 2.0**-20
                  + (2.0**-8 if rounded else 0.0)) * (p @ v.abs())
                 + 2.0**(5 - r) * v.abs().amax() + step * want.abs())
        worst = ((got[b, :, :n].double() - want).abs() - bound).max().item()
        assert worst <= 0.0, (b, p0, worst)


def filled(cuda, b, h, n, d, seed=0, std=1.0):
    cache = int8_kv(b, h, n, d, cuda)
    k, v = rows(b, n, h, d, seed, std=std), rows(b, n, h, d, seed + 1, std=std)
    int8_kv_append(cache, k.to(cuda), v.to(cuda), torch.zeros(1, dtype=torch.int64, device=cuda))
    return cache


def slopes_of(cuda, h):
    return torch.exp2(-torch.arange(1, h + 1, dtype=torch.float32, device=cuda))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("past", [0, 1, 15, 16, 62, 63, 64, 65, 200, 255, 300, 1000])
def test_single_tokens(cuda, past, d):
    print(f"int8 attention past={past} D={d}", flush=True)
    cache = filled(cuda, 2, 3, past + 1, d)
    q = rows(2, 1, 3, d, 7).to(cuda)
    for out_dtype in (None, torch.float32):
        check_attention(q, cache, torch.tensor([past], device=cuda), out_dtype=out_dtype)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("h,hkv", [(4, 4), (8, 1), (6, 2), (20, 1), (48, 2)])
@pytest.mark.parametrize("cap,biased", [(0.0, False), (15.0, False), (0.0, True), (15.0, True)])
def test_scores_and_shared_heads(cuda, h, hkv, cap, biased, d):
    print(f"int8 attention H={h}/{hkv} cap={cap} {biased} D={d}", flush=True)
    cache = filled(cuda, 2, hkv, 333, d, std=2.0)
    q = rows(2, 1, h, d, 5, torch.float32, 3.0).to(cuda)
    slopes = slopes_of(cuda, h) if biased else None
    check_attention(q, cache, torch.tensor([332, 100], device=cuda), cap=cap, slopes=slopes)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new", [2, 3, 17, 31, 32, 33, 64, 65, 130, 300])
@pytest.mark.parametrize("h,hkv", [(3, 3), (6, 2)])
def test_several_tokens(cuda, new, h, hkv, d):
    print(f"int8 attention new={new} H={h}/{hkv} D={d}", flush=True)
    cache = filled(cuda, 3, hkv, 400, d)
    q = rows(3, new, h, d, 3).to(cuda)
    start = torch.tensor([0, 61, 400 - new], device=cuda)
    check_attention(q, cache, start, slopes=slopes_of(cuda, h))
    check_attention(q, cache, torch.tensor([77], device=cuda), cap=9.0, out_dtype=torch.float32)
    lengths = torch.tensor([new, 1, new - 1], device=cuda)
    check_attention(q, cache, start, lengths=lengths)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 5, 40])
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_negative_slopes(cuda, cap, new, d):
    print(f"int8 attention negative slopes new={new} cap={cap} D={d}", flush=True)
    cache = filled(cuda, 2, 3, 700, d)
    q = rows(2, new, 3, d, 7).to(cuda)
    start = torch.tensor([700 - new, 130], device=cuda)
    check_attention(q, cache, start, cap=cap, slopes=-slopes_of(cuda, 3))


def test_sequences_switched_off_and_positions_past_the_end(cuda):
    cache = filled(cuda, 4, 2, 128, 64)
    for new in (1, 40):
        q = rows(4, new, 2, 64).to(cuda)
        start = torch.tensor([100 - new, -1, 128, 5], device=cuda)
        lengths = torch.tensor([new, new, new, 0], device=cuda)
        out = int8_kv_attention(q, cache, start, lengths=lengths)
        assert bool(torch.isfinite(out[0]).all()) and not out[1].any() and not out[3].any()
        assert bool(out[2].isnan().all())
        check_attention(q[:1], Int8KV(*(t[:1] for t in cache)), start[:1])


def test_a_long_cache(cuda):
    """Scores that lie far apart between blocks, many splits."""
    cache = filled(cuda, 1, 2, 20000, 128, std=1.5)
    q = rows(1, 1, 4, 128, 9, torch.float32, 4.0).to(cuda)
    check_attention(q, cache, torch.tensor([19999], device=cuda))
    check_attention(q, cache, torch.tensor([19999], device=cuda), slopes=slopes_of(cuda, 4))


def test_tokens_behind_the_position_do_not_count(cuda):
    cache = filled(cuda, 1, 2, 256, 128)
    q = rows(1, 1, 2, 128, 9).to(cuda)
    start = torch.tensor([130], device=cuda)
    want = int8_kv_attention(q, cache, start)
    cache.keys[:, :, 2, 3:] = 127  # block 2 holds positions 128 .. 130
    cache.values[:, :, 2, :, 3:] = -127
    for t in (cache.key_scales, cache.value_scales):
        t[:, :, 3] = math.nan
    assert torch.equal(int8_kv_attention(q, cache, start), want)


def test_a_later_block_of_nan_scale_stays_with_the_queries_that_see_it(cuda):
    cache = filled(cuda, 1, 1, 128, 64)
    cache.value_scales[:, :, 1] = math.nan
    cache.key_scales[:, :, 1] = math.nan
    q = rows(1, 8, 1, 64).to(cuda)
    out = int8_kv_attention(q, cache, torch.tensor([60], device=cuda))
    assert bool(torch.isfinite(out[:, :, :4]).all()) and bool(out[:, :, 4:].isnan().all())


def test_layouts_of_the_operands(cuda):
    cache = filled(cuda, 2, 2, 100, 64)
    q = rows(2, 3, 4, 64, 3).to(cuda)
    start = torch.tensor([90], device=cuda)
    want = int8_kv_attention(q, cache, start)
    wide = torch.zeros(2, 4, 3, 67, device=cuda, dtype=q.dtype)[..., 2:66].copy_(q)
    for other in (q.contiguous(), wide, q.transpose(2, 3).contiguous().transpose(2, 3)):
        assert torch.equal(int8_kv_attention(other, cache, start), want)
    half = int8_kv_attention(q.half(), cache, start)
    assert half.dtype == torch.float16
    k = torch.zeros(2, 2, 3, 67, device=cuda, dtype=q.dtype)[..., 2:66].copy_(q[:, :2])
    one, two = int8_kv(2, 2, 100, 64, cuda), int8_kv(2, 2, 100, 64, cuda)
    int8_kv_append(one, k, k, start)
    int8_kv_append(two, q[:, :2].half(), q[:, :2].half(), start)
    for a, b in zip(one, two):
        assert torch.equal(a, b)  # these bf16 values are fp16 numbers too
    big = int8_kv_read(cache, 0, 99, torch.bfloat16)
    for a, b in zip(big, int8_kv_read(cache, 0, 99)):
        assert torch.equal(a, b.to(torch.bfloat16))


def test_captured_steps(cuda):
    """Append and attention of a step in one graph, the position advanced on the device; two
    graphs of the same cache replayed in turn, each replay against an eager twin."""
    b, h, d = 3, 2, 128
    caches = [filled(cuda, b, h, 512, d) for _ in range(2)]
    q, k, v = (rows(b, 1, h, d, i).to(cuda) for i in range(3))
    pos = torch.tensor([50, 126, -1], device=cuda)

    def step(cache):
        int8_kv_append(cache, k, v, pos)
        return int8_kv_attention(q, cache, pos, softcap=20.0)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(caches[0])
        step(caches[1])
    torch.cuda.current_stream().wait_stream(stream)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(caches[0])
        graphs.append((graph, out))
    for i in range(6):
        for t, seed in ((q, 1), (k, 2), (v, 3)):
            t.copy_(rows(b, 1, h, d, 100 * i + seed, std=0.5 + i))
        graph, out = graphs[i % 2]
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, step(caches[1]))
        for x, y in zip(*caches):
            assert torch.equal(x, y)
        pos += 1


def test_refusals(cuda):
    cache = int8_kv(2, 2, 100, 64, cuda)
    q = torch.zeros(2, 4, 1, 64, device=cuda)
    start = torch.zeros(1, dtype=torch.int64, device=cuda)
    assert cache.capacity == 128
    with pytest.raises(ValueError, match="head sizes"):
        int8_kv(1, 1, 10, 80, cuda)
    with pytest.raises(ValueError, match="positive"):
        int8_kv(1, 0, 10, 64, cuda)
    with pytest.raises(RuntimeError, match="requires CUDA"):
        int8_kv(1, 1, 10, 64, "cpu")
    with pytest.raises(ValueError, match="shape"):
        int8_kv_append(cache, q, q, start)
    with pytest.raises(TypeError, match="dtype"):
        int8_kv_append(cache, q[:, :2], q[:, :2].double(), start)
    with pytest.raises(ValueError, match="start must be int64"):
        int8_kv_append(cache, q[:, :2], q[:, :2], start.int())
    with pytest.raises(ValueError, match="start must be int64"):
        int8_kv_attention(q, cache, start.expand(3))
    with pytest.raises(ValueError, match="lengths must be int64"):
        int8_kv_attention(q, cache, start, lengths=start)
    with pytest.raises(ValueError, match="device"):
        int8_kv_attention(q, cache, start.cpu())
    with pytest.raises(ValueError, match="heads"):
        int8_kv_attention(q[:, :3], cache, start)
    with pytest.raises(ValueError, match="softcap"):
        int8_kv_attention(q, cache, start, softcap=-1.0)
    with pytest.raises(ValueError, match="1e-3"):
        int8_kv_attention(q, cache, start, softcap=1e4)
    with pytest.raises(RuntimeError, match="no gradient"):
        int8_kv_attention(q.clone().requires_grad_(), cache, start)
    with pytest.raises(ValueError, match="past the cache"):
        int8_kv_read(cache, 0, 129)
    with pytest.raises(RuntimeError, match="contiguous"):
        ratchet().int8_kv_read(cache.keys.transpose(0, 1), *cache[1:], 0, 1, torch.float32)


def test_opcheck(cuda):
    cache = filled(cuda, 2, 2, 100, 64)
    x = rows(2, 3, 2, 64).to(cuda)
    start = torch.tensor([90], device=cuda)
    ops = ratchet()
    torch.library.opcheck(ops.int8_kv_append, (x, x, *cache, start, None))
    torch.library.opcheck(ops.int8_kv_read, (*cache, 3, 70, torch.float32))
    torch.library.opcheck(ops.int8_kv_attention, (x, *cache, start, None, 0.125, 5.0, None,
                                                  torch.bfloat16))
