"""Causal attention whose scores are capped, biased by the distance and masked by documents.

``causal_attention`` (``attention.py``) is the attention of the reference model
(``model.py:117-123``): every position sees all earlier ones, with the scores as they are. Here
the scores may be modified, each change on its own or together:

    s_ij = scale q_i . k_j
    s_ij = softcap tanh(s_ij / softcap)           softcap given
    s_ij = s_ij - slopes[h] |i - j|               slopes given, one per query head
    o_i  = sum_j softmax_j(s_ij) v_j              over the keys that i sees

and a mask (``attention_mask``) says what a query sees: its own document up to itself, and the
whole of the marked prefix its document begins with. A query that sees nothing gets zeros, and
sends and receives no gradient. k and v may have fewer heads than q (``H % Hkv == 0``; query head
h reads key head ``h // (H // Hkv)``).

On the GPU, bfloat16 with head size 64 or 128 runs on HIP kernels forward and backward
(``csrc/rk_scored.hip``, ``csrc/rk_scored_bwd.hip``); operands that do not lie as 16-byte rows
are copied first. Other types, head sizes and devices, and caps outside 1e-3 .. 1e3 (whose scores
the kernels' exponentials do not resolve), take the same formulas in torch operations (float32,
float64 for float64 operands), which hold all [B, H, S, S] scores at once.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch
from torch import Tensor

from .ops import ratchet


class AttentionMask(NamedTuple):
    """The plan of a mask, made once per batch by ``attention_mask`` and shared by the layers.

    ``bounds`` [4, B, S] int32: the keys ``bounds[0] <= j < bounds[1]`` that a query sees and the
    queries ``bounds[2] <= i < bounds[3]`` that see a key (zeros for padding); ``padding``
    [B, ceil(S / 32)] int32: a bit per position. B may be 1 for a mask all sequences share."""

    bounds: Tensor
    padding: Tensor


def attention_mask(documents: Tensor | None = None, prefix: Tensor | None = None
                   ) -> AttentionMask:
    """The mask of ``documents`` [B, S] (integers) and ``prefix`` [B, S] (bool), either or both.

    A document is a run of equal ids >= 0 (an id that comes back later begins another one);
    negative ids are padding, which sees nothing and is seen by nothing, whatever its keys and
    values hold. Without ``documents`` a row is one document. Positions see their document up to
    themselves, and the run of marked positions their document begins with (marks behind that run
    do not count)."""
    if documents is None and prefix is None:
        raise ValueError("attention_mask needs documents or prefix")
    for name, t in (("documents", documents), ("prefix", prefix)):
        if t is not None and t.dim() != 2:
            raise ValueError(f"{name} must be [B, S]")
    if documents is not None and (documents.is_floating_point() or documents.is_complex()
                                  or documents.dtype == torch.bool):
        raise TypeError("documents must hold integers")
    if prefix is not None and prefix.dtype != torch.bool:
        raise TypeError("prefix must be a bool tensor")
    if documents is not None and prefix is not None:
        if documents.shape != prefix.shape:
            raise ValueError("documents and prefix must share a [B, S] shape")
        if documents.device != prefix.device:
            raise ValueError("documents and prefix must share a device")
    if documents is not None and documents.dtype not in (torch.int32, torch.int64):
        documents = documents.to(torch.int64)
    like = documents if documents is not None else prefix
    if like.is_cuda:
        return AttentionMask(*ratchet().attention_mask(documents, prefix))
    return _torch_mask(documents, prefix)


def _torch_mask(documents: Tensor | None, prefix: Tensor | None) -> AttentionMask:
    like = documents if documents is not None else prefix
    b, s = like.shape
    at = torch.arange(s, device=like.device).expand(b, s)
    ids = documents if documents is not None else torch.zeros_like(at)
    first = torch.ones_like(ids, dtype=torch.bool)
    first[:, 1:] = ids[:, 1:] != ids[:, :-1]
    begin = torch.where(first, at, 0).cummax(1).values if s else at
    lead = torch.zeros_like(first)
    if prefix is not None and s:
        lead = torch.where(prefix, -1, at).cummax(1).values < begin

    def next_at(here: Tensor) -> Tensor:
        """The least later position where `here` holds, or s."""
        least = torch.where(here, at, s).flip(1).cummin(1).values.flip(1) if s else at
        return torch.cat([least[:, 1:], torch.full_like(least[:, :1], s)], dim=1)

    rows = [begin, torch.where(lead, next_at(first | ~lead), at + 1),
            torch.where(lead, begin, at), next_at(first)]
    bounds = torch.where(ids >= 0, torch.stack(rows), 0).to(torch.int32)
    bits = torch.zeros(b, -(-s // 32) * 32, dtype=torch.int64, device=like.device)
    bits[:, :s] = ids < 0
    words = (bits.view(b, -(-s // 32), 32) << torch.arange(32, device=like.device)).sum(-1)
    return AttentionMask(bounds, torch.where(words >= 2**31, words - 2**32, words).to(torch.int32))


def torch_scores(q: Tensor, k: Tensor, v: Tensor, seen: Tensor, distance: Tensor,
                 softcap: float, slopes: Tensor | None, scale: float) -> Tensor:
    """The formulas in torch operations, in float32 (float64 for float64 operands): `seen` and
    `distance` broadcast to the scores [B, H, Q, K]."""
    with torch.autocast(q.device.type, enabled=False):
        work = torch.float64 if q.dtype == torch.float64 else torch.float32
        group = q.shape[1] // k.shape[1] if k.shape[1] else 1
        kk, vv = (t.to(work).repeat_interleave(group, dim=1) for t in (k, v))
        scores = q.to(work) @ kk.transpose(2, 3).contiguous() * scale
        if softcap:
            scores = softcap * torch.tanh(scores / softcap)
        if slopes is not None:
            scores = scores - slopes.to(work)[:, None, None] * distance
        weights = scores.masked_fill(~seen, -math.inf)
        weights = torch.where(seen.any(-1, keepdim=True), weights, 0.0).softmax(-1)
        return (weights.masked_fill(~seen, 0.0) @ vv).to(q.dtype)


def _torch_scored_attention(q: Tensor, k: Tensor, v: Tensor, mask: AttentionMask | None,
                            softcap: float, slopes: Tensor | None, scale: float) -> Tensor:
    at = torch.arange(q.shape[2], device=q.device)
    if mask is None:
        seen = at[None, :] <= at[:, None]
    else:
        seen = ((at >= mask.bounds[0][..., None]) & (at < mask.bounds[1][..., None]))[:, None]
        # padding may hold anything: its products are masked, its values are cleared here
        used = (mask.bounds[1] > mask.bounds[0])[:, None, :, None]
        q, k, v = (torch.where(used, t, 0) for t in (q, k, v))
    return torch_scores(q, k, v, seen, (at[:, None] - at[None, :]).abs(), softcap, slopes, scale)


def score_arguments(q: Tensor, softcap: float | None, slopes: Tensor | None,
                    scale: float | None) -> tuple[float, Tensor | None, float]:
    """(softcap or 0, float32 slopes, scale) checked against q [B, H, S, D]."""
    softcap = 0.0 if softcap is None else float(softcap)
    if not 0.0 <= softcap < math.inf:
        raise ValueError("softcap must be finite and not negative")
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError("scale must be positive and finite")
    if slopes is not None:
        if slopes.shape != (q.shape[1],):
            raise ValueError("slopes must hold one value per query head")
        if not slopes.is_floating_point():
            raise TypeError("slopes must be floating point")
        if slopes.device != q.device:
            raise ValueError("slopes must be on the queries' device")
        slopes = slopes.float()
    return softcap, slopes, scale


def scored_attention(q: Tensor, k: Tensor, v: Tensor, *, mask: AttentionMask | None = None,
                     softcap: float | None = None, slopes: Tensor | None = None,
                     scale: float | None = None) -> Tensor:
    """Attention of q [B, H, S, D] over k, v [B, Hkv, S, D] with modified scores (see the module).

    ``mask``: from ``attention_mask`` (None: causal). ``softcap``: the scores' bound (None or 0:
    none). ``slopes`` [H]: the bias per step of distance (differentiable). ``scale``: default
    1 / sqrt(D). Returns [B, H, S, D] in q's dtype. The kernels have first derivatives in reverse
    mode; second ones and operands with a forward-mode tangent are refused."""
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape:
        raise ValueError("scored_attention expects q [B, H, S, D] and k, v [B, Hkv, S, D]")
    b, h, s, d = q.shape
    if (k.shape[0], k.shape[2], k.shape[3]) != (b, s, d) or d == 0:
        raise ValueError("q, k and v must agree in batch, length and head size")
    if k.shape[1] == 0 and h > 0 or k.shape[1] > 0 and h % k.shape[1] != 0:
        raise ValueError("query heads must be a multiple of the key heads")
    if not q.dtype == k.dtype == v.dtype or not q.is_floating_point():
        raise TypeError("q, k and v must share a floating-point dtype")
    if not q.device == k.device == v.device:
        raise ValueError("q, k and v must share a device")
    softcap, slopes, scale = score_arguments(q, softcap, slopes, scale)
    if mask is not None:
        rows = mask.bounds.shape[1] if mask.bounds.dim() == 3 else -1
        if mask.bounds.shape != (4, rows, s) or rows not in (1, b):
            raise ValueError("the mask must hold one row or one per sequence, of q's length")
        if mask.bounds.device != q.device:
            raise ValueError("the mask must be on the queries' device")
    if (q.is_cuda and q.dtype == torch.bfloat16 and d in (64, 128)
            and (softcap == 0.0 or 1e-3 <= softcap <= 1e3)):
        bounds, padding = mask if mask is not None else (None, None)
        return ratchet().scored_attend(q, k, v, bounds, padding, slopes, softcap, scale)
    return _torch_scored_attention(q, k, v, mask, softcap, slopes, scale)
