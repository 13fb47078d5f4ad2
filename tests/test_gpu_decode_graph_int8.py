"""Captured decode steps over an 8-bit cache where the step runs through the module forwards, and
behind work that is still queued."""

from __future__ import annotations

import pytest
import torch

from local_ai_training.decode import fused_decode_supported
from local_ai_training.generate import DecodeGraph, generate
from local_ai_training.model import ModelConfig, build_seeded_model

pytestmark = pytest.mark.gpu

SCORES = {"attention_softcap": 20.0, "distance_bias": True}


def model_of(cuda, mode="int8", max_code=2, **kw):
    config = ModelConfig(vocab_size=64, block_size=160, n_layer=2, n_head=2, n_embd=128,
                         ffn_hidden=256, matmul_mode=mode, **kw)
    return build_seeded_model(config, max_code=max_code, seed=3).to(cuda).eval()


def tokens_of(cuda, b, s):
    return torch.randint(0, 64, (b, s), generator=torch.Generator().manual_seed(s)).to(cuda)


@pytest.mark.parametrize("scores", [{}, SCORES])
@pytest.mark.parametrize("mode,max_code,b", [("bf16", 2, 2), ("fp32", 2, 2), ("fp32", None, 2),
                                             ("int8", 2, 17), ("int8", 2, 2)])
def test_steps_through_the_module_forwards(cuda, mode, max_code, b, scores):
    print(f"decode graph mode={mode} max_code={max_code} B={b} {bool(scores)}", flush=True)
    model = model_of(cuda, mode, max_code, **scores)
    model.fused_decode = mode != "int8" or b > 16  # the others are not fused by themselves
    tokens = tokens_of(cuda, b, 80)
    caches = [model.new_cache(b, dtype=torch.int8) for _ in range(2)]
    for cache in caches:
        model.prefill(tokens[:, :60], cache)
        assert not (model.fused_decode and fused_decode_supported(model, cache))
    kept = [t.clone() for layer in range(2) for t in caches[0].store(layer)]
    graph = DecodeGraph(model, caches[0])
    for a, t in zip(kept, (t for layer in range(2) for t in caches[0].store(layer))):
        assert torch.equal(a, t)
    for i in range(60, 70):
        got = graph.step(tokens[:, i:i + 1]).clone()
        torch.cuda.synchronize()
        want = model.decode_step(tokens[:, i:i + 1], caches[1])
        # the same products; a library may sum them in another order under a capture, and a code
        # then falls to the other side now and then
        assert (got.float() - want.float()).norm() <= 2.0**-6 * want.float().norm()
    assert int(caches[0].pos) == caches[0].length == 70


def test_a_graph_behind_a_queued_prompt(cuda):
    model = model_of(cuda, **SCORES)
    tokens = tokens_of(cuda, 2, 100)
    cache, twin = (model.new_cache(2, dtype=torch.int8) for _ in range(2))
    model.prefill(tokens[:, :90], twin)
    x = torch.randn(4096, 4096, device=cuda)
    torch.cuda.synchronize()
    for _ in range(40):  # some milliseconds of work ahead of the prompt
        x = (x @ x).clamp_(-1.0, 1.0)
    model.prefill(tokens[:, :90], cache)
    graph = DecodeGraph(model, cache)
    assert int(cache.pos) == cache.length == 90
    for i in range(90, 96):
        got = graph.step(tokens[:, i:i + 1]).clone()
        torch.cuda.synchronize()
        assert torch.equal(got, model.decode_step(tokens[:, i:i + 1], twin))


@pytest.mark.parametrize("mode,max_code", [("bf16", 2), ("fp32", None)])
def test_generate(cuda, mode, max_code):
    model = model_of(cuda, mode, max_code)
    letters = tuple(chr(48 + i) for i in range(64))
    text = generate(model, letters, "01234567", max_new_tokens=12, temperature=0.0,
                    cache_dtype=torch.int8, use_graph=True)
    assert len(text) == 12
