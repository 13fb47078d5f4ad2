"""A key/value cache in 8 bits on HIP kernels (``csrc/rk_kv8.hip``).

The bf16 cache of ``model.KVCache`` holds 4 bytes per feature of a token and head; this one holds
2, plus one float32 scale per 64 tokens for each of keys and values. A block's scale is its
largest absolute value / 127 and a code is ``rint(x / scale)``, so a value is off by at most half
a scale when it is written. Tokens appended to a block that holds some can raise its scale; its
codes are then rounded again, each time by at most half the scale of that time. A sequence ends
with the tokens appended last: positions behind them in their block no longer hold anything.

Positions are device tensors (int64, one for the batch or one per sequence), so steps have fixed
shapes and can be replayed as a HIP graph, and sequences may have different lengths. A negative
position switches a sequence off (nothing is appended, its attention is zeros); positions past
the cache are not written, and their attention is NaN.

The cache is GPU-only; the reference has none (``generate.py:183-201`` recomputes the window)."""

from __future__ import annotations

from typing import NamedTuple

import torch
import torch.autograd.forward_ad as forward_ad
from torch import Tensor

from .ops import ratchet
from .scored_attention import score_arguments

BLOCK = 64
HEAD_SIZES = (64, 128, 256)


class Int8KV(NamedTuple):
    """One layer's cache: ``keys`` int8 [B, H, blocks, 64, D], ``values`` int8
    [B, H, blocks, D, 64] (by feature, as the attention's second product reads them), scales
    float32 [B, H, blocks]."""

    keys: Tensor
    values: Tensor
    key_scales: Tensor
    value_scales: Tensor

    @property
    def capacity(self) -> int:
        return self.keys.shape[2] * BLOCK


def int8_kv(batch: int, heads: int, max_len: int, head_size: int,
            device: torch.device | str | int) -> Int8KV:
    """An empty cache of `max_len` positions (rounded up to whole blocks) for `heads` key heads."""
    if min(batch, heads, max_len) <= 0:
        raise ValueError("cache dimensions must be positive")
    if head_size not in HEAD_SIZES:
        raise ValueError(f"an 8-bit cache takes head sizes {HEAD_SIZES}")
    device = torch.device(device)
    if device.type != "cuda":
        raise RuntimeError("an 8-bit cache requires CUDA (a ROCm GPU)")
    blocks = -(-max_len // BLOCK)
    codes = dict(dtype=torch.int8, device=device)
    return Int8KV(torch.zeros(batch, heads, blocks, BLOCK, head_size, **codes),
                  torch.zeros(batch, heads, blocks, head_size, BLOCK, **codes),
                  torch.zeros(batch, heads, blocks, device=device),
                  torch.zeros(batch, heads, blocks, device=device))


def _check_positions(cache: Int8KV, start: Tensor, lengths: Tensor | None) -> None:
    batch = cache.keys.shape[0]
    for name, t, sizes in (("start", start, (1, batch)), ("lengths", lengths, (batch,))):
        if t is None:
            continue
        if t.dtype != torch.int64 or t.dim() != 1 or t.shape[0] not in sizes:
            raise ValueError(f"{name} must be int64, one per sequence" +
                             (" or one for the batch" if name == "start" else ""))
        if t.device != cache.keys.device:
            raise ValueError(f"{name} must be on the cache's device")


def _refuse_gradients(what: str, *operands: Tensor | None) -> None:
    for t in operands:
        if t is not None and ((t.requires_grad and torch.is_grad_enabled())
                              or forward_ad.unpack_dual(t).tangent is not None):
            raise RuntimeError(f"{what} an 8-bit cache has no gradient; call it under no_grad, "
                               "on operands without tangents")


def int8_kv_append(cache: Int8KV, k: Tensor, v: Tensor, start: Tensor,
                   lengths: Tensor | None = None) -> None:
    """Writes k and v [B, H, S, D] at positions ``start`` .. of each sequence; of a sequence's S
    tokens the first ``lengths`` count (None: all). It has no gradient."""
    b, h, _, _, d = cache.keys.shape
    if k.dim() != 4 or k.shape != v.shape or (k.shape[0], k.shape[1], k.shape[3]) != (b, h, d):
        raise ValueError("k and v must share the cache's [B, H, S, D] shape")
    if k.dtype != v.dtype or not k.is_floating_point():
        raise TypeError("k and v must share a floating-point dtype")
    _refuse_gradients("appending to", k, v)
    if not k.device == v.device == cache.keys.device:
        raise ValueError("k and v must be on the cache's device")
    _check_positions(cache, start, lengths)
    if k.dtype not in (torch.float32, torch.bfloat16):
        k, v = k.float(), v.float()
    ratchet().int8_kv_append(k.detach(), v.detach(), *cache, start.contiguous(),
                             lengths.contiguous() if lengths is not None else None)


def int8_kv_attention(q: Tensor, cache: Int8KV, start: Tensor, *, lengths: Tensor | None = None,
                      softcap: float | None = None, slopes: Tensor | None = None,
                      scale: float | None = None, out_dtype: torch.dtype | None = None) -> Tensor:
    """Attention of q [B, Hq, S, D] over the cache (Hq a multiple of its heads): query i of a
    sequence stands at position ``start`` + i and sees positions 0 .. ``start`` + i, which must
    have been appended. The score's cap, bias and scale are those of ``scored_attention``.
    Returns [B, Hq, S, D] in ``out_dtype`` (default q's); queries at or past ``lengths`` are
    zeros. It has no gradient."""
    b, h, _, _, d = cache.keys.shape
    if q.dim() != 4 or q.shape[0] != b or q.shape[3] != d or q.shape[1] % h:
        raise ValueError("q must be [B, Hq, S, D] with heads a multiple of the cache's")
    if not q.is_floating_point():
        raise TypeError("q must be floating point")
    _refuse_gradients("attention over", q, slopes)
    if q.device != cache.keys.device:
        raise ValueError("q must be on the cache's device")
    out_dtype = out_dtype or q.dtype
    if not out_dtype.is_floating_point:
        raise TypeError("out_dtype must be floating point")
    _check_positions(cache, start, lengths)
    softcap, slopes, scale = score_arguments(q, softcap, slopes, scale)
    if softcap and not 1e-3 <= softcap <= 1e3:
        raise ValueError("softcap must lie in 1e-3 .. 1e3")
    if q.dtype not in (torch.float32, torch.bfloat16):
        q = q.float()
    native = out_dtype if out_dtype in (torch.float32, torch.bfloat16) else torch.float32
    out = ratchet().int8_kv_attention(
        q, *cache, start.contiguous(), lengths.contiguous() if lengths is not None else None,
        scale, softcap, slopes.detach() if slopes is not None else None, native)
    return out if native == out_dtype else out.to(out_dtype)


def int8_kv_read(cache: Int8KV, begin: int = 0, end: int | None = None,
                 dtype: torch.dtype = torch.float32) -> tuple[Tensor, Tensor]:
    """The keys and values [B, H, end - begin, D] that positions begin .. end - 1 stand for."""
    end = cache.capacity if end is None else end
    if not 0 <= begin <= end <= cache.capacity:
        raise ValueError("positions past the cache")
    if dtype not in (torch.float32, torch.bfloat16):
        raise TypeError("values are read as float32 or bfloat16")
    return ratchet().int8_kv_read(*cache, begin, end, dtype)
