"""Drafted tokens judged in one pass, on HIP kernels (``csrc/rk_tree.hip``, ``csrc/rk_verify.hip``).

A small model or a lookup proposes a tree of tokens behind a sequence; the large model runs all of
them at once, and those that its own distribution would have drawn stand. The reference runs the
model once for every token (``generate.py:183-201``).

* ``draft_tree``: the plan of a tree, from its nodes' parents.
* ``tree_attention``: the nodes' attention over the 8-bit cache (``int8_cache.py``) and over the
  nodes on their own way from the root. Their keys and values lie beside the cache, so rejected ones
  never raise the scale of a block.
* ``verify_drafts``: the nodes that stand, and the token behind them. The tokens are distributed as
  the target model's own at that temperature and ``top_k``, whatever the drafts were.
* ``int8_kv_commit``: the keys and values of the nodes that stood, of all layers, into their caches.
* ``sample_tokens``: one token of each row of logits, by the same rules.

Node 0 is the root: the last token that is known, which the cache does not hold yet. A sequence with
``start`` cached tokens has its nodes at positions ``start`` + depth.
"""

from __future__ import annotations

import math
from typing import NamedTuple, Sequence

import torch
from torch import Tensor

from .int8_cache import Int8KV
from .ops import ratchet
from .scored_attention import torch_scores

MAX_NODES = 256
_NATIVE = (torch.float32, torch.bfloat16)
_NOTHING = 2.0**-40  # a residual of this sum is rounding


def check_batch(batch: int) -> None:
    if batch != 1:
        raise ValueError("a model's cache has one position for the batch: drafts of one sequence "
                         "can be committed to it (int8_kv_commit takes any)")


class DraftTree(NamedTuple):
    """The plan of trees, made by ``draft_tree``: one for all sequences or one for each (R 1 or B).

    ``parents`` [R, N] int32 (-1 for the root, -2 for nodes that are off), ``depths`` [R, N] int32
    (steps from the root), ``seen`` [R, N, ceil(N / 64)] int64: a bit for a node itself and for each
    of its ancestors, none for nodes that are off."""

    parents: Tensor
    depths: Tensor
    seen: Tensor


def draft_tree(parents: Tensor | Sequence[int], device: torch.device | str | None = None
               ) -> DraftTree:
    """The plan of the trees with these `parents`, [N] or [R, N] integers: -1 for node 0, an earlier
    node for every other one. Numbers on the host are checked; in a GPU tensor, which is not waited
    for, a node with another parent and all that descends from it are off (zeros in attention, never
    accepted). At most 256 nodes."""
    p = torch.as_tensor(parents)
    if p.is_floating_point() or p.is_complex() or p.dtype == torch.bool:
        raise TypeError("parents must be integers")
    if p.dim() == 1:
        p = p[None]
    if p.dim() != 2 or p.shape[1] == 0:
        raise ValueError("parents must be [N] or [R, N], with a root")
    n = p.shape[1]
    if n > MAX_NODES:
        raise ValueError(f"a tree has at most {MAX_NODES} nodes")
    if not p.is_cuda:
        at = torch.arange(n)
        if not bool(((p[:, 0] == -1) & ((p[:, 1:] >= 0) & (p[:, 1:] < at[1:])).all(1)).all()):
            raise ValueError("node 0 must have the parent -1, every other node an earlier one")
        tree = _torch_tree(p.tolist())
        return tree if device is None else DraftTree(*(t.to(device) for t in tree))
    if device is not None and p.device != torch.empty(0, device=device).device:
        raise ValueError("parents on a GPU are planned there")
    return DraftTree(*ratchet().draft_tree(p if p.dtype == torch.int32 else p.to(torch.int64)))


def _torch_tree(rows: list[list[int]]) -> DraftTree:
    depths, seen = [], []
    for parents in rows:
        depth, bits = [], []
        for i, parent in enumerate(parents):
            depth.append(depth[parent] + 1 if i else 0)
            bits.append(1 << i | (bits[parent] if i else 0))
        depths.append(depth)
        words = [[b >> 64 * w & 2**64 - 1 for w in range(-(-len(parents) // 64))] for b in bits]
        seen.append([[x - 2**64 if x >= 2**63 else x for x in row] for row in words])
    return DraftTree(torch.tensor(rows, dtype=torch.int32),
                     torch.tensor(depths, dtype=torch.int32),
                     torch.tensor(seen, dtype=torch.int64))


def _lineage(tree: DraftTree) -> Tensor:
    """Which node sees which, bool [R, N, N]."""
    r, n, _ = tree.seen.shape
    shifts = torch.arange(64, device=tree.seen.device)
    return (tree.seen[..., None] >> shifts & 1).bool().reshape(r, n, -1)[:, :, :n]


def tree_attention(q: Tensor, k: Tensor, v: Tensor, cache: Int8KV, start: Tensor,
                   tree: DraftTree, *, lengths: Tensor | None = None,
                   softcap: float | None = None, slopes: Tensor | None = None,
                   scale: float | None = None, out_dtype: torch.dtype | None = None) -> Tensor:
    """Attention of a tree's nodes, q [B, Hq, N, D] and k, v [B, H, N, D] (Hq a multiple of H, the
    cache's heads): node i stands at position ``start`` + depth and sees the cache's positions
    0 .. ``start`` - 1, its ancestors and itself. ``start`` as in ``int8_kv_attention`` (negative: a
    sequence that is off); of a sequence's nodes the first ``lengths`` [B] are there. The score's
    cap, bias (by the distance of the positions) and scale are those of ``scored_attention``.
    Returns [B, Hq, N, D] in ``out_dtype`` (default q's); zeros for nodes that are off or not there.
    Nothing is appended to the cache. It has no gradient."""
    if not (q.dtype == k.dtype == v.dtype and q.dtype in _NATIVE):
        for t in (q, k, v):
            if not t.is_floating_point():
                raise TypeError("q, k and v must be floating point")
        out_dtype = out_dtype or q.dtype
        q, k, v = q.float(), k.float(), v.float()
    out_dtype = out_dtype or q.dtype
    if not out_dtype.is_floating_point:
        raise TypeError("out_dtype must be floating point")
    native = out_dtype if out_dtype in _NATIVE else torch.float32
    if scale is None:
        scale = q.shape[-1] ** -0.5 if q.shape[-1] else 1.0
    out = ratchet().tree_attention.default(
        q, k, v, *cache, start, lengths, tree.depths, tree.seen, scale, softcap or 0.0, slopes,
        native)
    return out if native == out_dtype else out.to(out_dtype)


def torch_tree_attention(q: Tensor, k: Tensor, v: Tensor, keys: Tensor, values: Tensor,
                         start: int, tree: DraftTree, softcap: float, slopes: Tensor | None,
                         scale: float) -> Tensor:
    """The same over a cache of floats, keys and values [B, H, >= start, D], in torch operations."""
    n = q.shape[2]
    at = torch.arange(start, device=q.device)
    kin = _lineage(tree)
    seen = torch.cat([(kin.any(-1, keepdim=True)).expand(-1, n, start), kin], dim=2)
    depths = tree.depths[:, :, None]
    distance = torch.cat([start + depths - at, depths - tree.depths[:, None, :]], dim=2)
    joined = (torch.cat([c[:, :, :start], t.to(c.dtype)], dim=2)
              for c, t in ((keys, k), (values, v)))
    return torch_scores(q, *joined, seen[:, None], distance.abs()[:, None], softcap, slopes, scale)


class Verified(NamedTuple):
    """``path`` [B, N] int64: the nodes that stand, from the root on, then -1; ``counts`` [B]: how
    many; ``next`` [B]: the token behind the last of them."""

    path: Tensor
    counts: Tensor
    next: Tensor


def verify_drafts(logits: Tensor, tokens: Tensor, tree: DraftTree,
                  uniforms: Tensor | None = None, *, lengths: Tensor | None = None,
                  draft_logits: Tensor | None = None, temperature: float = 1.0,
                  top_k: int | None = None) -> Verified:
    """Which of a tree's drafted `tokens` [B, N] stand, from the target's `logits` [B, N, V] at its
    nodes (of the token that follows each) and random numbers `uniforms` [B, N] in [0, 1).

    With p, q the softmax of the target's and the drafter's logits at a node over ``temperature``,
    without logits below the ``top_k``-th largest: the node's children are tried in their order; one of
    token x stands if u q(x) < p(x), otherwise p becomes max(p - q, 0) over its sum (but for sums up to
    2^-40, of drafts that q does not hold: then p stays). Where none stands, the next token is the first
    whose cumulated p passes the root's u times its sum. The children of a node must have been drawn
    from q independently; without ``draft_logits`` each counts as certain (drafts from a lookup, or the
    drafter's best). At temperature 0 a child stands if its token is the target's first largest logit's.

    Of a sequence's nodes the first ``lengths`` [B] are there (none: count 0, next -1); a child whose
    token is outside 0 .. V - 1 is taken as not there. A row that is
    no distribution (a NaN, +inf, only -inf) gives next -1 (at temperature 0 a NaN is the largest, as
    in torch's argmax). Decisions are made in 64 bits. Logits of other
    types than float32 and bfloat16 are taken as float32."""
    if logits.dtype not in _NATIVE or (draft_logits is not None
                                       and draft_logits.dtype != logits.dtype):
        for t in (logits, draft_logits):
            if t is not None and not t.is_floating_point():
                raise ValueError("logits must be floating point")
        logits = logits.float()
        draft_logits = draft_logits.float() if draft_logits is not None else None
    if top_k is not None and top_k <= 0:
        raise ValueError("top_k must be positive")
    if logits.is_cuda:
        if logits.requires_grad or (draft_logits is not None and draft_logits.requires_grad):
            logits = logits.detach()
            draft_logits = draft_logits.detach() if draft_logits is not None else None
        return Verified(*ratchet().verify_drafts.default(
            logits, tokens, tree.parents, uniforms, lengths, draft_logits, temperature,
            top_k or 0))
    _check_verification(logits, tokens, tree, uniforms, lengths, draft_logits, temperature)
    with torch.no_grad():
        return _torch_verify(logits, tokens, tree, uniforms, lengths, draft_logits, temperature,
                             top_k or 0)


def _check_verification(logits: Tensor, tokens: Tensor, tree: DraftTree,
                        uniforms: Tensor | None, lengths: Tensor | None,
                        draft_logits: Tensor | None, temperature: float) -> None:
    """The operator's own checks, for the torch form."""
    if logits.dim() != 3 or logits.shape[1] == 0 or logits.shape[2] == 0:
        raise ValueError("logits must be [B, N, V], of at least the root")
    b, n, _ = logits.shape
    if tokens.shape != (b, n) or tokens.dtype != torch.int64:
        raise ValueError("tokens must be int64 [B, N]")
    if not (temperature == 0.0 or 1e-6 <= temperature < math.inf):
        raise ValueError("temperature must be finite and at least 1e-6 (0: greedy)")
    if temperature and uniforms is None:
        raise ValueError("sampling needs uniforms")
    if uniforms is not None and (uniforms.shape != (b, n) or uniforms.dtype != torch.float32):
        raise ValueError("uniforms must be float32 [B, N]")
    if draft_logits is not None and draft_logits.shape != logits.shape:
        raise ValueError("the drafter's logits must have the target's shape")
    if lengths is not None and (lengths.shape != (b,) or lengths.dtype != torch.int64):
        raise ValueError("lengths must be int64, one per sequence")
    for t in (tokens, uniforms, draft_logits, lengths, *tree):
        if t is not None and t.device != logits.device:
            raise ValueError("the operands must share a device")
    rows = tree.parents.shape[0]
    if rows not in (1, b) or tree.parents.shape != (rows, n):
        raise ValueError("the tree must hold one row or one per sequence, of these nodes")


def _distribution(row: Tensor, temperature: float, top_k: int) -> Tensor:
    x = row.double()
    if top_k and top_k < x.shape[0]:
        x = x.masked_fill(x < x.topk(top_k).values[-1], -math.inf)
    return (x / temperature).softmax(0)


def _torch_verify(logits: Tensor, tokens: Tensor, tree: DraftTree, uniforms: Tensor | None,
                  lengths: Tensor | None, draft_logits: Tensor | None, temperature: float,
                  top_k: int) -> Verified:
    b, n, vocab = logits.shape
    path = torch.full((b, n), -1, dtype=torch.int64, device=logits.device)
    counts, following = [], []
    for s in range(b):
        parents = tree.parents[s % tree.parents.shape[0]].tolist()
        there = n if lengths is None else min(int(lengths[s]), n)
        if there <= 0 or parents[0] != -1:
            counts.append(0)
            following.append(-1)
            continue
        way, pick = [0], -1
        p = q = None
        for i in range(there):
            if i and parents[i] != way[-1]:
                continue
            token = int(tokens[s, i])
            if i == 0:
                stands = True
            elif temperature == 0.0:
                stands = token == pick
            else:
                known = 0 <= token < vocab
                if draft_logits is None:
                    q = torch.zeros_like(p)
                    if known:
                        q[token] = 1.0
                stands = known and float(uniforms[s, i]) * float(q[token]) < float(p[token])
                if not stands and known:
                    left = (p - q).clamp(min=0.0) if draft_logits is not None else p * (q == 0)
                    total = left.sum()
                    p = p if total <= _NOTHING else left / total
            if stands:
                way += [i] if i else []
                row = logits[s, i]
                if temperature == 0.0:
                    pick = int(row.argmax())
                else:
                    p = _distribution(row, temperature, top_k)
                    if draft_logits is not None:
                        q = _distribution(draft_logits[s, i], temperature, top_k)
        if temperature != 0.0:
            sums = p.cumsum(0)
            pick = -1
            if bool(sums[-1] > 0.0):
                over = torch.nonzero(sums > float(uniforms[s, 0]) * sums[-1])
                pick = int(over[0]) if over.numel() else int(torch.nonzero(p > 0.0)[-1])
        path[s, :len(way)] = torch.tensor(way, device=path.device)
        counts.append(len(way))
        following.append(pick)
    as_ints = dict(dtype=torch.int64, device=logits.device)
    return Verified(path, torch.tensor(counts, **as_ints), torch.tensor(following, **as_ints))


def sample_tokens(logits: Tensor, uniforms: Tensor | None = None, *, temperature: float = 1.0,
                  top_k: int | None = None) -> Tensor:
    """One token for each row of `logits` [B, V], int64 [B]: the first whose cumulated probability
    passes `uniforms` [B] (at temperature 0 the first largest logit's). Rows that are no
    distribution give -1."""
    if logits.dim() != 2:
        raise ValueError("logits must be [B, V]")
    if uniforms is not None and uniforms.shape != logits.shape[:1]:
        raise ValueError("uniforms must hold one number per row")
    root = torch.zeros(logits.shape[0], 1, dtype=torch.int64, device=logits.device)
    one = torch.full((1, 1), -1, dtype=torch.int32, device=logits.device)
    tree = DraftTree(one, one + 1, one.to(torch.int64)[..., None] + 2)
    return verify_drafts(logits[:, None], root, tree,
                         uniforms[:, None] if uniforms is not None else None,
                         temperature=temperature, top_k=top_k).next


def int8_kv_commit(caches: Sequence[Int8KV], ks: Sequence[Tensor], vs: Sequence[Tensor],
                   start: Tensor, path: Tensor, counts: Tensor) -> None:
    """Appends accepted nodes to every layer's cache, in one launch for 32 layers: token i <
    ``counts`` [B] of a sequence is node ``path`` [B, P] [i] of the layer's k and v [B, H, N, D], and
    goes to position ``start`` + i (as ``int8_kv_append`` puts it there). Nodes outside 0 .. N - 1
    within the counts are tokens of zeros. It has no gradient."""
    if not ks or not len(caches) == len(ks) == len(vs):
        raise ValueError("one k, one v and one cache per layer are needed")
    if ks[0].dtype not in _NATIVE and ks[0].is_floating_point():
        ks, vs = [k.float() for k in ks], [v.float() for v in vs]
    ratchet().int8_kv_commit.default(ks, vs, *zip(*caches), start, path, counts)
