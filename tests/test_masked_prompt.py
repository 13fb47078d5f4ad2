"""What may follow a prompt under a mask, on the CPU: behind one document (and its prefix) the cache
goes on as the window does; behind several documents or padding, which later positions must not
see and the cache does not tell apart, every way on is refused."""

from __future__ import annotations

import pytest
import torch

from local_ai_training.generate import DecodeGraph
from local_ai_training.model import ModelConfig, build_seeded_model
from local_ai_training.scored_attention import attention_mask


def model_of(**kw):
    config = ModelConfig(vocab_size=40, block_size=48, n_layer=2, n_head=2, n_embd=32, **kw)
    return build_seeded_model(config, max_code=None, seed=1).eval()


def prompt():
    return torch.randint(0, 40, (2, 20), generator=torch.Generator().manual_seed(3))


@pytest.mark.parametrize("kw", [{}, {"attention_softcap": 2.0, "distance_bias": True}])
@pytest.mark.parametrize("ids", [False, True])
def test_a_prefix_goes_on_as_the_window_does(kw, ids):
    model, tokens = model_of(**kw), prompt()
    prefix = torch.zeros(2, 20, dtype=torch.bool)
    prefix[0, :5] = prefix[1, :8] = True
    documents = torch.tensor([[4], [0]]).expand(2, 20) if ids else None

    def mask(n):
        return attention_mask(documents[:, :n] if ids else None, prefix[:, :n])

    want = model(tokens, mask=mask(20))[0]
    cache = model.new_cache(2)
    got = [model.prefill(tokens[:, :9], cache, mask=mask(9)),
           model.prefill(tokens[:, 9:13], cache)]
    got += [model.decode_step(tokens[:, i:i + 1], cache) for i in range(13, 20)]
    for logits, i in zip(got, [8, 12, *range(13, 20)]):
        # float32 sums in another order, logits of order one
        assert torch.allclose(logits, want[:, i], rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("kind", ["documents", "padding behind", "padding before"])
def test_other_masks_end_the_cache(kind):
    model, tokens = model_of(), prompt()
    documents = torch.zeros(2, 9, dtype=torch.int64)
    documents[1] = {"documents": torch.tensor([0] * 8 + [1]),
                    "padding behind": torch.tensor([0] * 8 + [-1]),
                    "padding before": torch.tensor([-1] + [0] * 8)}[kind]
    cache = model.new_cache(2, max_len=12)
    logits = model.prefill(tokens[:, :9], cache, mask=attention_mask(documents))
    assert logits.shape == (2, 40) and cache.length == 9
    with pytest.raises(ValueError, match="several documents or padding"):
        model.decode_step(tokens[:, 9:10], cache)
    with pytest.raises(ValueError, match="several documents or padding"):
        model.prefill(tokens[:, 9:11], cache)
    with pytest.raises(ValueError, match="several documents or padding"):
        DecodeGraph(model, cache)
    with pytest.raises(ValueError, match="start of the cache"):
        model.prefill(tokens[:, 9:11], cache, mask=attention_mask(documents[:, :2]))
    with pytest.raises(ValueError, match="full"):
        model.prefill(tokens[:, 9:13], cache)
    assert cache.length == int(cache.pos) == 9
    cache.length = 0  # started anew, without a mask
    cache.pos.zero_()
    want = model(tokens[:, :10])[0]
    model.prefill(tokens[:, :9], cache)
    got = model.decode_step(tokens[:, 9:10], cache)
    assert torch.allclose(got, want[:, 9], rtol=1e-4, atol=1e-5)
