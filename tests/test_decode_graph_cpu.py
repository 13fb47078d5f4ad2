"""What building a decode graph does before it captures, on the CPU with the GPU's streams and
graphs replaced by nothing: the step is warmed up at a position that exists, and the position of
an 8-bit cache is neither moved nor read back from another stream."""

from __future__ import annotations

import contextlib

import pytest
import torch

from local_ai_training import model as model_module
from local_ai_training.generate import DecodeGraph
from local_ai_training.int8_cache import Int8KV
from local_ai_training.model import Int8KVCache, KVCache, ModelConfig, build_seeded_model


class _Stream:
    def __init__(self, *args, **kw):
        pass

    def wait_stream(self, other):
        pass


@pytest.fixture
def no_gpu(monkeypatch):
    for name in ("Stream", "current_stream"):
        monkeypatch.setattr(torch.cuda, name, _Stream)
    monkeypatch.setattr(torch.cuda, "CUDAGraph", object)
    for name in ("stream", "graph"):
        monkeypatch.setattr(torch.cuda, name, lambda *args, **kw: contextlib.nullcontext())

    def store(batch, heads, max_len, head, device):
        n = -(-max_len // 64)
        return Int8KV(torch.zeros(batch, heads, n, 64, head, dtype=torch.int8),
                      torch.zeros(batch, heads, n, head, 64, dtype=torch.int8),
                      torch.zeros(batch, heads, n), torch.zeros(batch, heads, n))

    def init(self, *shape):
        KVCache.__init__(self, *shape, torch.int8)
        self.stores = [None] * self.n_layer

    monkeypatch.setattr(model_module, "int8_kv", store)
    monkeypatch.setattr(Int8KVCache, "__init__", init)


@pytest.mark.parametrize("mode,max_code", [("fp32", 2), ("fp32", None)])
@pytest.mark.parametrize("greedy", [False, True])
def test_the_warm_up_of_a_model_that_is_not_fused(no_gpu, monkeypatch, mode, max_code, greedy):
    config = ModelConfig(vocab_size=16, block_size=32, n_layer=2, n_head=1, n_embd=64,
                         matmul_mode=mode)
    model = build_seeded_model(config, max_code=max_code, seed=0).eval()
    model.blocks = torch.nn.ModuleList()  # embedding, positions and head are left
    monkeypatch.setattr("local_ai_training.generate.decode_greedy", lambda *args: None)
    cache = model.new_cache(3, dtype=torch.int8)
    cache.advance(5)
    version = cache.pos._version
    graph = DecodeGraph(model, cache, greedy=greedy)
    assert graph.logits.shape == (3, 16)
    assert int(cache.pos) == cache.length == 5
    # moved and moved back on a side stream, its value would hang on the order of two streams
    assert cache.pos._version == version
    # nothing is left for the capture to allocate and clear
    assert all(s is not None for s in cache.stores)
