"""The 8-bit cache has no gradients: whatever operand wants one (or has a forward-mode tangent) is
refused before anything runs, instead of being left out of it."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from local_ai_training.int8_cache import Int8KV, int8_kv_append, int8_kv_attention


def operands():
    cache = Int8KV(torch.zeros(1, 2, 1, 64, 64, dtype=torch.int8),
                   torch.zeros(1, 2, 1, 64, 64, dtype=torch.int8),
                   torch.zeros(1, 2, 1), torch.zeros(1, 2, 1))
    return cache, torch.zeros(1, 2, 1, 64), torch.zeros(1, dtype=torch.int64)


@pytest.fixture
def untouched(monkeypatch):
    """No call may reach the library."""
    def reached():
        raise AssertionError("the library was called")
    monkeypatch.setattr("local_ai_training.int8_cache.ratchet", reached)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_slopes(untouched, dtype):
    cache, x, start = operands()
    slopes = torch.ones(2, dtype=dtype, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        int8_kv_attention(x, cache, start, slopes=slopes)
    with torch.no_grad(), pytest.raises(AssertionError, match="library"):
        int8_kv_attention(x, cache, start, slopes=slopes)
    with pytest.raises(AssertionError, match="library"):
        int8_kv_attention(x, cache, start, slopes=slopes.detach())


@pytest.mark.parametrize("which", [0, 1])
def test_appended_keys_and_values(untouched, which):
    cache, x, start = operands()
    rows = [x, x]
    rows[which] = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        int8_kv_append(cache, *rows, start)
    with torch.no_grad(), pytest.raises(AssertionError, match="library"):
        int8_kv_append(cache, *rows, start)


@pytest.mark.parametrize("grad_mode", [True, False])
def test_tangents(untouched, grad_mode):
    cache, x, start = operands()
    with torch.set_grad_enabled(grad_mode), forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        slopes = forward_ad.make_dual(torch.ones(2), torch.ones(2))
        with pytest.raises(RuntimeError, match="no gradient"):
            int8_kv_attention(dual, cache, start)
        with pytest.raises(RuntimeError, match="no gradient"):
            int8_kv_attention(x, cache, start, slopes=slopes)
        for rows in ((dual, x), (x, dual)):
            with pytest.raises(RuntimeError, match="no gradient"):
                int8_kv_append(cache, *rows, start)
