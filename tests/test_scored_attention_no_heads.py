"""Attention with modified scores without query heads: keys and values that no query reads have
gradients of zero from the operator, and the C backward refuses the call, whose dk and dv it would
leave as they were."""

from __future__ import annotations

import ctypes

import pytest
import torch

from local_ai_training import _native as nat
from local_ai_training.scored_attention import attention_mask, scored_attention


class Args(ctypes.Structure):
    """rk_scored_attention_args"""
    _fields_ = ([(n, ctypes.c_void_p) for n in
                 "q k v o lse rest bounds padding slopes g dq dk dv dslopes".split()]
                + [(n, ctypes.c_int64) for n in "B H Hkv S D mask_batch".split()]
                + [("strides", ctypes.c_int64 * 21)]
                + [(n, ctypes.c_float) for n in ("scale", "softcap")])


def test_the_c_backward_refuses():
    lib = nat.load_library()
    args = Args(B=1, H=0, Hkv=2, S=8, D=64, scale=1.0)
    assert lib.rk_scored_attention_forward(ctypes.byref(args), None) == 0
    assert lib.rk_scored_attention_backward(ctypes.byref(args), None, None) == 1
    assert b"query heads" in lib.rk_last_error()
    for name in ("B", "Hkv", "S"):  # nothing to write
        empty = Args(B=1, H=0, Hkv=2, S=8, D=64, scale=1.0)
        setattr(empty, name, 0)
        assert lib.rk_scored_attention_backward(ctypes.byref(empty), None, None) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_gradients_of_keys_that_no_query_reads(cuda, d, masked):
    mask = attention_mask(torch.zeros(2, 40, dtype=torch.int64, device=cuda)) if masked else None
    k, v = (torch.randn(2, 3, 40, d, device=cuda).to(torch.bfloat16).requires_grad_()
            for _ in range(2))
    q = torch.zeros(2, 0, 40, d, device=cuda, dtype=torch.bfloat16, requires_grad=True)
    slopes = torch.zeros(0, device=cuda, requires_grad=True)
    out = scored_attention(q, k, v, mask=mask, slopes=slopes)
    junk = [torch.full_like(k, 3.0) for _ in range(8)]  # what freed memory would hold
    del junk
    dq, dk, dv, ds = torch.autograd.grad(out.float().sum(), [q, k, v, slopes])
    assert out.shape == dq.shape == q.shape and ds.shape == (0,)
    assert not dk.any() and not dv.any()
