"""Tree attention behind more positions than float32 numbers one by one (2^24): distances stay whole."""

from __future__ import annotations

import pytest
import torch

import draft_reference as plain
from local_ai_training.drafts import draft_tree, tree_attention
from local_ai_training.int8_cache import int8_kv, int8_kv_append, int8_kv_read

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def rows(cuda, h, n, seed, dtype):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(1, h, n, 64, generator=gen).to(dtype).to(cuda)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("past", [2**24 - 1, 2**24 + 1, 2**24 + 2])
def test_biased_scores_of_far_positions(cuda, past, dtype):
    """Slopes of 1 and 1/2: of the tokens further than 300 positions away, zeros, nothing is left (less
    than e^-140), so the plain form over the last 300 is the result's. Tolerance: a score is off by
        (D + 4) 2^-24 scale sum |q_f k_f| + 2^-21 (|raw| + |s| + bias),
    a probability by twice that, sums by 2 (T / 64 + 96) roundings of 2^-24 for the T blocks' tokens that
    weigh, probabilities by 2^-16 and the result by half a step for bf16."""
    print(f"far positions {past} {dtype}", flush=True)
    window, nodes = 300, 6
    cache = int8_kv(1, 1, 2**24 + 64, 64, cuda)
    k, v = rows(cuda, 1, window, 1, BF16), rows(cuda, 1, window, 2, BF16)
    int8_kv_append(cache, k, v, torch.tensor([past - window], device=cuda))
    q = rows(cuda, 2, nodes, 3, dtype)
    nk, nv = (rows(cuda, 1, nodes, seed, dtype) for seed in (4, 5))
    slopes, parents = torch.tensor([1.0, 0.5]), [-1, 0, 0, 1, 3, 4]
    got = tree_attention(q, nk, nv, cache, torch.tensor([past], device=cuda),
                         draft_tree(parents, cuda), slopes=slopes.to(cuda))
    keys, values = (t.double().cpu()[0] for t in int8_kv_read(cache, past - window, past))
    want, size, delta = plain.tree_attention(
        *(t[0].double().cpu() for t in (q, nk, nv)), keys, values, window, parents, 0.0,
        slopes.double(), 0.125)
    few = 2.0**-16 if dtype == BF16 else 2.0**-24
    bound = ((2 * delta + 2 * (window / 64 + 96) * 2.0**-24 + few) * size
             + torch.finfo(dtype).eps / 2 * want.abs())
    assert ((got[0].double().cpu() - want).abs() <= bound).all()
