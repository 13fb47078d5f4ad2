"""The model on packed documents with capped and biased scores, trained and then served from the
8-bit cache: the operators as they are used together."""

from __future__ import annotations

import math

import pytest
import torch

from local_ai_training import model as model_module
from local_ai_training import scored_attention as scored_module
from local_ai_training.generate import DecodeGraph, generate
from local_ai_training.int8_cache import int8_kv_attention, int8_kv_read
from local_ai_training.model import Int8KVCache, ModelConfig, build_seeded_model
from local_ai_training.scored_attention import attention_mask

pytestmark = pytest.mark.gpu

SCORES = {"attention_softcap": 20.0, "distance_bias": True}


def model_of(cuda, mode="int8", max_code=2, head=64, **kw):
    config = ModelConfig(vocab_size=64, block_size=160, n_layer=2, n_head=2, n_embd=2 * head,
                         ffn_hidden=256, matmul_mode=mode, int8_backward=mode == "int8", **kw)
    return build_seeded_model(config, max_code=max_code, seed=3).to(cuda)


def batch(cuda, b=2, s=130):
    gen = torch.Generator().manual_seed(s)
    tokens = torch.randint(0, 64, (b, s), generator=gen)
    documents = (torch.rand(b, s, generator=gen) < 0.03).cumsum(1)
    documents[-1, s - 20:] = -1
    prefix = torch.rand(b, s, generator=gen) < 0.3
    targets = tokens.roll(-1, 1).masked_fill(documents < 0, -100)
    return tokens.to(cuda), targets.to(cuda), attention_mask(documents.to(cuda), prefix.to(cuda))


@pytest.mark.parametrize("scores", [{}, SCORES])
def test_documents_do_not_see_each_other(cuda, scores):
    model = model_of(cuda, **scores).eval()
    tokens, _, _ = batch(cuda)
    documents = torch.zeros_like(tokens)
    documents[:, 70:] = 1
    mask = attention_mask(documents)
    other = tokens.clone()
    other[:, :70] = (other[:, :70] + 1) % 64
    with torch.no_grad(), torch.autocast("cuda", torch.bfloat16):
        first, second = model(tokens, mask=mask)[0], model(other, mask=mask)[0]
    assert torch.equal(first[:, 70:], second[:, 70:])
    assert not torch.equal(first[:, :70], second[:, :70])


def test_gradients_of_a_packed_step(cuda, monkeypatch):
    """The float model's gradients under bf16 autocast with the kernels, and with the torch form
    in float32 in their place. Each layer's attention differs by the rounding of p (2^-9 of a norm)
    and, backward, of ds, p and the results (2^-8 of a norm at most): two layers forward and
    backward move a gradient by at most 4 2^-8 of its norm, twice that with the layers' gain."""
    tokens, targets, mask = batch(cuda)
    grads = []
    for kernels in (True, False):
        model = model_of(cuda, mode="fp32", max_code=None, **SCORES).train()
        if not kernels:
            def plain(q, k, v, *, mask, softcap, slopes):
                return scored_module._torch_scored_attention(q, k, v, mask, softcap, slopes,
                                                             1.0 / math.sqrt(q.shape[-1]))
            monkeypatch.setattr(model_module, "scored_attention", plain)
        with torch.autocast("cuda", torch.bfloat16):
            _, loss = model(tokens, targets, mask=mask)
        loss.backward()
        grads.append([p.grad for p in model.parameters()])
    for a, b in zip(*grads):
        assert bool(torch.isfinite(a).all())
        assert (a - b).norm() <= 8 * 2.0**-8 * b.norm()


def test_a_ratchet_training_step_runs(cuda):
    model = model_of(cuda, **SCORES).train()
    tokens, targets, mask = batch(cuda)
    before = [m.packed.clone() for m in model.modules() if hasattr(m, "packed")]
    with torch.autocast("cuda", torch.bfloat16):
        _, loss = model(tokens, targets, mask=mask)
    loss.backward()
    model.ratchet_update()
    after = [m.packed for m in model.modules() if hasattr(m, "packed")]
    assert math.isfinite(loss.item())
    assert any(not torch.equal(a, b) for a, b in zip(before, after))
    assert bool(torch.isfinite(model.token_embedding.weight.grad).all())


@pytest.mark.parametrize("head", [64, 128, 256])
@pytest.mark.parametrize("scores", [{}, SCORES])
def test_cached_steps(cuda, scores, head):
    """A prompt and single tokens: the fused decode kernels and the module forwards read and
    write the same cache, and what it holds is the layers' keys and values to half a scale."""
    tokens, _, _ = batch(cuda, 3, 100)
    logits = []
    for fused in (True, False):
        model = model_of(cuda, head=head, **scores).eval()
        model.fused_decode = fused
        cache = model.new_cache(3, dtype=torch.int8)
        assert isinstance(cache, Int8KVCache)
        steps = [model.prefill(tokens[:, :60], cache)]
        steps += [model.decode_step(tokens[:, i:i + 1], cache) for i in range(60, 70)]
        steps.append(model.prefill(tokens[:, 70:], cache))  # a chunk behind what is cached
        logits.append((steps, cache))
    (a, cache), (b, other) = logits
    assert cache.length == other.length == 100 and int(cache.pos) == 100
    assert torch.equal(a[0], b[0])
    # the module path's attention output goes through the same row quantization; the sums
    # around it differ in order, logits are bfloat16 numbers
    for x, y in zip(a, b):
        assert (x - y).norm() <= 2.0**-6 * y.norm()
    window = model_of(cuda, head=head, **scores).eval()
    seen = {}
    hook = window.blocks[0].attention.qkv.register_forward_hook(
        lambda m, i, out: seen.setdefault("qkv", out))
    with torch.no_grad():
        window(tokens)
    hook.remove()
    qkv = seen["qkv"]
    parts = qkv if isinstance(qkv, tuple) else qkv.chunk(3, dim=-1)
    for got, want, scales in zip(int8_kv_read(cache.store(0), 0, 100), parts[1:],
                                 (cache.store(0).key_scales, cache.store(0).value_scales)):
        want = want.float().view(3, 100, 2, head).transpose(1, 2)
        # ten single tokens may each have rounded the block's codes again
        half = 0.5 * scales.repeat_interleave(64, dim=2)[:, :, :100, None]
        assert bool(((got - want).abs() <= 12 * half).all())
        assert bool(((got - want).abs()[:, :, 70:] <= 1.001 * half[:, :, 70:]).all())


def test_a_prompt_is_cached_to_half_a_scale_and_read(cuda):
    model = model_of(cuda, **SCORES).eval()
    tokens, _, mask = batch(cuda, 2, 130)
    cache = model.new_cache(2, max_len=140, dtype=torch.int8)
    a = model.prefill(tokens, cache, mask=mask)
    assert bool(torch.isfinite(a).all())
    with pytest.raises(ValueError, match="start of the cache"):
        model.prefill(tokens[:, :2], cache, mask=mask)
    with pytest.raises(ValueError, match="full"):
        model.prefill(tokens[:, :11], cache)
    with pytest.raises(TypeError, match="store"):
        cache.buffers(0, tokens)
    q = torch.randn(2, 2, 1, 64, device=cuda)
    out = int8_kv_attention(q, cache.store(1), cache.pos - 1)
    assert bool(torch.isfinite(out).all())


@pytest.mark.parametrize("scores", [{}, SCORES])
def test_a_captured_decode_step(cuda, scores):
    tokens, _, _ = batch(cuda, 2, 120)
    model = model_of(cuda, **scores).eval()
    caches = [model.new_cache(2, dtype=torch.int8) for _ in range(2)]
    for cache in caches:
        model.prefill(tokens[:, :57], cache)
    kept = [t.clone() for t in caches[0].store(1)]
    graph = DecodeGraph(model, caches[0])
    for a, b in zip(kept, caches[0].store(1)):
        assert torch.equal(a, b)  # neither warm-up nor capture touch the cache
    for i in range(57, 75):
        got = graph.step(tokens[:, i:i + 1]).clone()
        torch.cuda.synchronize()
        assert torch.equal(got, model.decode_step(tokens[:, i:i + 1], caches[1]))
    for a, b in zip(caches[0].store(1), caches[1].store(1)):
        assert torch.equal(a, b)
    greedy = DecodeGraph(model, caches[0], greedy=True)
    greedy.tokens.copy_(tokens[:, 75:76])
    picked = tokens[:, 75:76]
    for _ in range(4):
        got = greedy.next_greedy().clone()
        picked = model.decode_step(picked, caches[1]).argmax(-1, keepdim=True)
        assert torch.equal(got, picked)


def test_generate_from_the_8_bit_cache(cuda):
    model = model_of(cuda, **SCORES).eval()
    letters = tuple(chr(48 + i) for i in range(64))
    texts = [generate(model, letters, "01234567", max_new_tokens=12, temperature=0.0,
                      cache_dtype=torch.int8, use_graph=graph) for graph in (False, True)]
    assert len(texts[0]) == 12 and texts[0] == texts[1]
    assert len(generate(model, letters, "0123", max_new_tokens=3, temperature=0.0)) == 3
