"""Capped, biased and masked attention in the model on the CPU: documents do not see each other, a
float cache gives what the whole window gives, and what is refused."""

from __future__ import annotations

import pytest
import torch

from local_ai_training.model import ModelConfig, TransformerBlock, build_seeded_model
from local_ai_training.scored_attention import attention_mask


def model_of(**kw):
    config = ModelConfig(vocab_size=40, block_size=48, n_layer=2, n_head=2, n_embd=32, **kw)
    return build_seeded_model(config, max_code=None, seed=1).eval()


def test_documents_and_prefixes():
    model = model_of(attention_softcap=4.0, distance_bias=True)
    gen = torch.Generator().manual_seed(0)
    tokens = torch.randint(0, 40, (2, 30), generator=gen)
    documents = torch.zeros(2, 30, dtype=torch.int64)
    documents[:, 12:] = 1
    prefix = torch.zeros(2, 30, dtype=torch.bool)
    prefix[:, 12:16] = True
    mask = attention_mask(documents, prefix)
    first = model(tokens, mask=mask)[0]
    other = tokens.clone()
    other[:, :12] = (other[:, :12] + 1) % 40
    assert torch.equal(model(other, mask=mask)[0][:, 12:], first[:, 12:])
    other = tokens.clone()
    other[:, 15] = (other[:, 15] + 1) % 40  # seen by its prefix, unlike a later token
    assert bool((model(other, mask=mask)[0][:, 12] != first[:, 12]).any())
    other = tokens.clone()
    other[:, 20] = (other[:, 20] + 1) % 40
    changed = model(other, mask=mask)[0]
    assert torch.equal(changed[:, :20], first[:, :20])


@pytest.mark.parametrize("kw", [{"attention_softcap": 2.0}, {"distance_bias": True},
                                {"attention_softcap": 2.0, "distance_bias": True}])
def test_a_float_cache_follows_the_window(kw):
    model = model_of(**kw)
    tokens = torch.randint(0, 40, (3, 20), generator=torch.Generator().manual_seed(1))
    want = model(tokens)[0]
    cache = model.new_cache(3)
    got = [model.prefill(tokens[:, :7], cache)]
    got.append(model.prefill(tokens[:, 7:12], cache))
    got += [model.decode_step(tokens[:, i:i + 1], cache) for i in range(12, 20)]
    for logits, i in zip(got, [6, 11, *range(12, 20)]):
        # float32 sums in another order, logits of order one
        assert torch.allclose(logits, want[:, i], rtol=1e-4, atol=1e-5)
    plain = model_of()
    assert not torch.allclose(plain(tokens)[0], want, atol=1e-3)


def test_checkpointed_blocks_take_the_mask():
    tokens = torch.randint(0, 40, (2, 16), generator=torch.Generator().manual_seed(2))
    mask = attention_mask(torch.arange(16).div(5, rounding_mode="floor").expand(2, -1))
    grads = []
    for checkpointing in (False, True):
        model = model_of(gradient_checkpointing=checkpointing, distance_bias=True).train()
        _, loss = model(tokens, tokens, mask=mask)
        loss.backward()
        grads.append([p.grad for p in model.parameters()])
    for a, b in zip(*grads):
        assert torch.equal(a, b)


def test_the_state_dict_is_the_plain_model_s():
    assert model_of(distance_bias=True).state_dict().keys() == model_of().state_dict().keys()


def test_refusals():
    with pytest.raises(ValueError, match="softcap"):
        model_of(attention_softcap=-1.0)
    with pytest.raises(ValueError, match="dropout"):
        model_of(distance_bias=True, dropout=0.1)
    model = model_of()
    with pytest.raises(RuntimeError, match="requires CUDA"):
        model.new_cache(1, dtype=torch.int8)
    tokens = torch.zeros(1, 4, dtype=torch.int64)
    mask = attention_mask(torch.zeros(1, 4, dtype=torch.int64))
    cache = model.new_cache(1)
    model.prefill(tokens, cache, mask=mask)
    with pytest.raises(ValueError, match="start of the cache"):
        model.prefill(tokens, cache, mask=mask)
    config = ModelConfig(vocab_size=8, n_embd=32, n_head=2, dropout=0.5)
    block = TransformerBlock(config, max_code=None).train()
    with pytest.raises(ValueError, match="dropout"):
        block(torch.zeros(1, 4, 32), mask=mask)
