"""A masked prompt and the 8-bit cache: what the layers append lies within half a scale of their
keys and values, the prompt's logits are those of the masked window, steps behind it are the same
through the fused kernels, the module forwards and a captured graph, and the attention over what the cache
holds is that of the values read back."""

from __future__ import annotations

import math

import pytest
import torch

from local_ai_training.generate import DecodeGraph
from local_ai_training.int8_cache import int8_kv_attention, int8_kv_read
from local_ai_training.model import ModelConfig, build_seeded_model
from local_ai_training.scored_attention import attention_mask

pytestmark = pytest.mark.gpu

SCORES = {"attention_softcap": 20.0, "distance_bias": True}


def model_of(cuda, **kw):
    config = ModelConfig(vocab_size=64, block_size=160, n_layer=2, n_head=2, n_embd=128,
                         ffn_hidden=256, matmul_mode="int8", **kw)
    return build_seeded_model(config, max_code=2, seed=3).to(cuda).eval()


def tokens_of(cuda, s):
    return torch.randint(0, 64, (2, s), generator=torch.Generator().manual_seed(s)).to(cuda)


def prefix_mask(cuda, s):
    prefix = torch.zeros(2, s, dtype=torch.bool, device=cuda)
    prefix[0, :40] = prefix[1, :90] = True
    return attention_mask(prefix=prefix)


@pytest.mark.parametrize("scores", [{}, SCORES])
@pytest.mark.parametrize("kind", ["prefix", "documents"])
def test_a_prompt_is_appended_to_half_a_scale(cuda, kind, scores):
    model, s = model_of(cuda, **scores), 130
    tokens = tokens_of(cuda, s)
    mask = prefix_mask(cuda, s)
    if kind == "documents":
        mask = attention_mask((torch.arange(s, device=cuda) // 60).expand(2, s))
    appended = [[], []]
    hooks = [block.attention.qkv.register_forward_hook(
        lambda m, i, out, kept=kept: kept.append(out)) for block, kept in
        zip(model.blocks, appended)]
    cache = model.new_cache(2, max_len=140, dtype=torch.int8)
    logits = model.prefill(tokens, cache, mask=mask)
    for hook in hooks:
        hook.remove()
    for layer, kept in enumerate(appended):
        parts = kept[0] if isinstance(kept[0], tuple) else kept[0].chunk(3, dim=-1)
        store = cache.store(layer)
        for got, x, scales in zip(int8_kv_read(store, 0, s), parts[1:],
                                  (store.key_scales, store.value_scales)):
            x = x.float().view(2, s, 2, 64).transpose(1, 2)
            # code x scale and the code's quotient are float32 roundings, 2^-16 of a step at 127
            half = (0.5 + 2.0**-15) * scales.repeat_interleave(64, dim=2)[:, :, :s, None]
            assert bool(((got - x).abs() <= half).all())
    # a bfloat16 cache attends to the same operands under the same mask; the window's projections
    # are float32, its logits bfloat16 numbers a few roundings of 2^-8 away
    caches = [model.new_cache(2, max_len=140, dtype=torch.bfloat16) for _ in range(2)]
    assert torch.equal(logits, model.prefill(tokens, caches[0], mask=mask))
    assert not torch.equal(logits, model.prefill(tokens, caches[1]))
    with torch.no_grad():
        want = model(tokens, mask=mask)[0][:, -1]
    assert (logits - want).float().norm() <= 2.0**-5 * want.float().norm()
    q = torch.randn(2, 2, 1, 64, device=cuda)
    keys, values = (t.double() for t in int8_kv_read(cache.store(1), 0, s))
    p = (q.double() @ keys.transpose(2, 3).contiguous() / math.sqrt(64)).softmax(-1)
    got = int8_kv_attention(q, cache.store(1), cache.pos - 1)
    # float32 results; scores of order ten off by 2^-21 of themselves
    assert bool(((got.double() - p @ values).abs() <= 2.0**-15 * (p @ values.abs())).all())


@pytest.mark.parametrize("scores", [{}, SCORES])
def test_steps_behind_a_prefix(cuda, scores):
    tokens = tokens_of(cuda, 120)
    runs = []
    for way in ("fused", "modules", "graph"):
        model = model_of(cuda, **scores)
        model.fused_decode = way != "modules"
        cache = model.new_cache(2, dtype=torch.int8)
        model.prefill(tokens[:, :100], cache, mask=prefix_mask(cuda, 100))
        graph = DecodeGraph(model, cache) if way == "graph" else None
        steps = []
        for i in range(100, 110):
            token = tokens[:, i:i + 1]
            steps.append((graph.step(token) if graph else model.decode_step(token, cache)).clone())
        runs.append(steps)
        assert int(cache.pos) == cache.length == 110
    for fused, modules, captured in zip(*runs):
        assert torch.equal(fused, captured)
        # sums in another order, logits are bfloat16 numbers
        assert (fused - modules).norm() <= 2.0**-6 * modules.norm()


def test_a_cache_that_cannot_go_on(cuda):
    model, tokens = model_of(cuda), tokens_of(cuda, 120)
    documents = torch.zeros(2, 100, dtype=torch.int64, device=cuda)
    documents[1, 90:] = -1
    cache = model.new_cache(2, dtype=torch.int8)
    model.prefill(tokens[:, :100], cache, mask=attention_mask(documents))
    for go_on in (lambda: model.decode_step(tokens[:, 100:101], cache),
                  lambda: model.prefill(tokens[:, 100:105], cache),
                  lambda: DecodeGraph(model, cache)):
        with pytest.raises(ValueError, match="several documents or padding"):
            go_on()
