"""Commits of drafts without a node: an accepted token of them would have nothing to be."""

from __future__ import annotations

import ctypes

import pytest
import torch

from local_ai_training import _native as nat
from local_ai_training.drafts import int8_kv_commit
from local_ai_training.int8_cache import Int8KV

_i64, _p = ctypes.c_int64, ctypes.c_void_p


def cache_of(b=2, h=2, blocks=1, d=64):
    return Int8KV(torch.zeros(b, h, blocks, 64, d, dtype=torch.int8),
                  torch.zeros(b, h, blocks, d, 64, dtype=torch.int8),
                  torch.zeros(b, h, blocks), torch.zeros(b, h, blocks))


def test_no_nodes():
    none = torch.zeros(2, 2, 0, 64)
    with pytest.raises(ValueError, match="root"):
        int8_kv_commit([cache_of()], [none], [none], torch.zeros(1, dtype=torch.int64),
                       torch.zeros(2, 3, dtype=torch.int64), torch.ones(2, dtype=torch.int64))


class CommitLayer(ctypes.Structure):
    """rk_int8_kv_commit_layer."""

    _fields_ = [*((name, _p) for name in ("keys", "values", "key_scales", "value_scales")),
                *((name, _i64) for name in ("B", "H", "blocks", "D")), ("k", _p), ("v", _p),
                *((name, _i64) for name in ("skb", "skh", "sks", "svb", "svh", "svs"))]


def test_no_nodes_at_the_c_entry():
    fake = 1 << 12  # never dereferenced
    layer = CommitLayer(keys=fake, values=fake, key_scales=fake, value_scales=fake, B=1, H=1, blocks=1,
                        D=64, k=fake, v=fake)
    lib = nat.load_library()
    args = (_i64(1), _i64(0), 0, _p(fake), _i64(1), _p(fake), _i64(3))
    assert lib.rk_int8_kv_commit(ctypes.byref(layer), *args, _i64(3), _p(fake), None) == 1
    assert b"no nodes" in lib.rk_last_error()
    # no path: nothing to append
    assert lib.rk_int8_kv_commit(ctypes.byref(layer), *args, _i64(0), _p(fake), None) == 0
