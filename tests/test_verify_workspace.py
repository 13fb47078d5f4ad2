"""The verification's C entries on the host: workspace of sizes that the call itself refuses."""

from __future__ import annotations

import ctypes

import pytest

from local_ai_training import _native as nat

_i64, _p = ctypes.c_int64, ctypes.c_void_p


class VerifyArgs(ctypes.Structure):
    """rk_verify_drafts_args."""

    _fields_ = [("logits", _p), ("drafts", _p),
                *((name, _i64) for name in ("lb", "ln", "db", "dn", "B", "N", "V", "trees", "top_k")),
                ("tokens", _p), ("uniforms", _p), ("parents", _p), ("lengths", _p),
                ("temperature", ctypes.c_double), ("path", _p), ("counts", _p), ("next", _p),
                ("dtype", ctypes.c_int)]


def args_of(b, n, v, temperature):
    fake = 1 << 12  # never dereferenced
    return VerifyArgs(logits=fake, tokens=fake, uniforms=fake, parents=fake, path=fake, counts=fake,
                      next=fake, B=b, N=n, V=v, trees=1, temperature=temperature)


@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_workspace_of_what_a_launch_holds(temperature):
    lib = nat.load_library()
    for b, n, v in ((1, 1, 1), (3, 5, 300), (2, 256, 70000), (1 << 21, 1, 9)):
        args = args_of(b, n, v, temperature)
        assert lib.rk_verify_drafts_work(ctypes.byref(args)) >= 24 * 2 * b * n


@pytest.mark.parametrize("temperature", [0.0, 1.0])
@pytest.mark.parametrize("b,n,v,message", [
    (1, 1, 0, b"empty vocabulary"), (1, 1, -5, b"negative"), (1, 257, 5, b"256 nodes"),
    (1 << 32, 1, 5, b"too many"), (1 << 56, 256, 5, b"too many"), (1 << 20, 256, 5, b"too many")])
def test_workspace_of_sizes_that_are_refused(b, n, v, message, temperature):
    """A caller asks for the workspace before the call says what is wrong: nothing is needed."""
    lib = nat.load_library()
    args = args_of(b, n, v, temperature)
    assert lib.rk_verify_drafts_work(ctypes.byref(args)) == 0
    assert lib.rk_verify_drafts(ctypes.byref(args), None, _i64(0), None) != 0
    assert message in lib.rk_last_error()


def test_workspace_of_nothing():
    lib = nat.load_library()
    for b, n in ((0, 5), (5, 0)):
        args = args_of(b, n, 7, 1.0)
        assert lib.rk_verify_drafts_work(ctypes.byref(args)) == 0
        assert lib.rk_verify_drafts(ctypes.byref(args), None, _i64(0), None) == 0
    assert lib.rk_verify_drafts_work(None) == 0
