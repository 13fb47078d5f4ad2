"""Drafted generation over the 8-bit key/value cache: what a program that lets a small model (or a
lookup) propose a tree of tokens, and the large one judge them all in one pass, has these operators
do.

Kinds of case:

* ``tree``: attention of the tree's nodes over the cache and over the nodes on their own way from
  the root, whose keys and values are not in the cache yet. Trees that differ from sequence to
  sequence are planned within the pass.
* ``verify``: which drafted tokens stand, given the target's logits at every node and random
  numbers, and the token that follows the last one that does.
* ``commit``: the keys and values of the nodes that stood, of all layers, into the layers' caches,
  and the touched blocks read back.

Head counts and sizes are those of the 25M (8 layers, 8 heads of 64, window 512) and the 1B
transformer (24 layers, 16 heads of 128, window 1024, vocabulary 8192) that the benchmark and the
tests run, or generic.

Definitions. A tree's node 0 is its root, the last token that is known; every other node's parent
comes before it. A sequence of `start` cached tokens has its nodes at positions start + depth; a node
sees the cached tokens, its ancestors and itself. The score is scale q.k, then cap tanh(. / cap),
then minus slope_h times the distance of the positions. Of a sequence's nodes the first `count` are
there; the others' results are zeros.

p_n and q_n are the softmax of the target's and the drafter's logits at node n over the temperature,
without what lies below the k-th largest logit (equal ones stay). The nodes are walked in order. At
node n a child c with token x stands if u_c q(x) < p(x), and the walk goes on from it; otherwise
p becomes max(p - q, 0) over its sum and the next child is tried. Without the drafter's logits q is
1 at the drafted token. Where no child stands, the next token is the first whose cumulated p passes
u_0 times its sum. At temperature 0 a child stands if its token is the target's first largest.

A cache block's scale is its largest absolute value / 127 and a code is rint(x / scale). Appended
tokens can only raise the scale s of a block that already holds tokens: to
max(s, largest new value / 127); its codes c are then rounded again, rint(c (s / s_new)). Scales,
quotients and ratios are float32 numbers, so the codes are defined to the last one.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False  # False: the plain forms; True: the framework's kernels

BLOCK = 64  # tokens of a cache block


def listed():
    return [
        # the 25M model, one sequence, a short chain of drafts: latency counts
        {"name": "tree_chain_25m", "kind": "tree", "batch": 1, "heads": 8, "kv_heads": 8,
         "head": 64, "past": 300, "ragged": False, "nodes": 5, "branch": 1, "cap": 0.0,
         "slopes": False, "type": "bf16"},
        # the 1B model near the end of its window, a tree of three drafts a node
        {"name": "tree_1b", "kind": "tree", "batch": 1, "heads": 16, "kv_heads": 16,
         "head": 128, "past": 980, "ragged": False, "nodes": 26, "branch": 3, "cap": 0.0,
         "slopes": False, "type": "bf16"},
        # a batch of long sequences of several lengths, a tree of its own for each
        {"name": "tree_b16_long", "kind": "tree", "batch": 16, "heads": 16, "kv_heads": 16,
         "head": 128, "past": 8000, "ragged": True, "nodes": 32, "branch": 0, "cap": 0.0,
         "slopes": False, "type": "bf16"},
        # long sequences, shared key heads, capped scores, large trees
        {"name": "tree_shared_64", "kind": "tree", "batch": 8, "heads": 32, "kv_heads": 4,
         "head": 64, "past": 16000, "ragged": True, "nodes": 64, "branch": 2, "cap": 30.0,
         "slopes": False, "type": "bf16"},
        # a distance bias, queries and results in float32, an odd number of nodes
        {"name": "tree_bias_f32", "kind": "tree", "batch": 4, "heads": 16, "kv_heads": 16,
         "head": 128, "past": 3001, "ragged": True, "nodes": 13, "branch": 2, "cap": 0.0,
         "slopes": True, "type": "f32"},
        # greedy generation with drafts from a lookup, a vocabulary of bytes: latency counts
        {"name": "verify_greedy_bytes", "kind": "verify", "batch": 1, "nodes": 8, "branch": 1,
         "vocab": 256, "type": "f32", "drafter": False, "temperature": 0.0, "top_k": 0},
        # the 1B model's vocabulary, one sequence, a sampled tree
        {"name": "verify_tree_1b", "kind": "verify", "batch": 1, "nodes": 26, "branch": 3,
         "vocab": 8192, "type": "f32", "drafter": True, "temperature": 0.8, "top_k": 40},
        # many sequences, sampled chains, an odd vocabulary
        {"name": "verify_chain_b64", "kind": "verify", "batch": 64, "nodes": 6, "branch": 1,
         "vocab": 32003, "type": "f32", "drafter": True, "temperature": 1.0, "top_k": 0},
        # drafts without a drafter's probabilities, a tree of its own for each sequence
        {"name": "verify_lookup_b8", "kind": "verify", "batch": 8, "nodes": 40, "branch": 0,
         "vocab": 50000, "type": "bf16", "drafter": False, "temperature": 0.7, "top_k": 50},
        # large trees over a large vocabulary
        {"name": "verify_tree_b16", "kind": "verify", "batch": 16, "nodes": 64, "branch": 4,
         "vocab": 131072, "type": "bf16", "drafter": True, "temperature": 1.0, "top_k": 0},
        # the 1B model's layers, one sequence
        {"name": "commit_1b", "kind": "commit", "layers": 24, "batch": 1, "kv_heads": 16,
         "head": 128, "start": 900, "nodes": 26, "branch": 3},
        # the 25M model's layers, many sequences
        {"name": "commit_25m_b32", "kind": "commit", "layers": 8, "batch": 32, "kv_heads": 8,
         "head": 64, "start": 445, "nodes": 40, "branch": 1},
    ]


def _between(rng, low, high):
    """An integer spread over the logarithm of its range."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "verify", "verify", "commit"])
    nodes, branch = _between(rng, 1, 64), rng.choice([0, 1, 2, 3, 4])
    if kind == "tree":
        batch, kv_heads = _between(rng, 1, 32), rng.choice([1, 2, 4, 8, 16])
        heads = kv_heads * rng.choice([1, 1, 2, 4, 8])
        # at most the largest listed case's keys times nodes
        longest = max(64, min(16000, 16 * 16 * 8000 // (batch * heads)))
        return {"kind": kind, "batch": batch, "heads": heads, "kv_heads": kv_heads,
                "head": rng.choice([64, 128]), "past": rng.choice([0, _between(rng, 1, longest)]),
                "ragged": rng.random() < 0.5, "nodes": nodes, "branch": branch,
                "cap": rng.choice([0.0, rng.uniform(5.0, 50.0)]),
                "slopes": rng.random() < 0.5, "type": rng.choice(["bf16", "bf16", "f32"])}
    if kind == "verify":
        vocab = _between(rng, 65, 131072)
        batch = _between(rng, 1, max(1, min(64, 16 * 64 * 131072 // (2 * nodes * vocab))))
        temperature = rng.choice([0.0, 1.0, rng.uniform(0.4, 1.5)])
        return {"kind": kind, "batch": batch, "nodes": nodes, "branch": branch, "vocab": vocab,
                "type": rng.choice(["f32", "bf16"]), "drafter": rng.random() < 0.6,
                "temperature": temperature, "top_k": rng.choice([0, _between(rng, 1, 200)])}
    return {"kind": kind, "layers": rng.randint(1, 24), "batch": _between(rng, 1, 8),
            "kv_heads": rng.choice([1, 2, 4, 8]), "head": rng.choice([64, 128]),
            "start": rng.randint(0, 900), "nodes": nodes, "branch": branch}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _trees(case):
    """Parents [rows][nodes] of a case (its own, whatever the seed): one row for a tree that all
    sequences share (branch children a node, level by level), one a sequence for branch 0, drawn
    among the last few nodes."""
    nodes, branch = case["nodes"], case["branch"]
    if branch:
        return [[-1] + [(i - 1) // branch for i in range(1, nodes)]]
    rng = random.Random(31 * nodes + case["batch"])
    return [[-1] + [rng.randint(max(0, i - 6), i - 1) for i in range(1, nodes)]
            for _ in range(case["batch"])]


def _counts(case):
    """How many nodes each sequence has: all, or, where each has its own tree, some."""
    if case["branch"]:
        return None
    rng = random.Random(case["nodes"] + 7 * case["batch"])
    return [rng.randint(max(1, case["nodes"] // 2), case["nodes"]) for _ in range(case["batch"])]


def _depths(parents):
    depths = []
    for parent in parents:
        depths.append(0 if parent < 0 else depths[parent] + 1)
    return depths


def _starts(case):
    """Cached tokens of each sequence (one number for all where they do not differ)."""
    if not case["ragged"]:
        return [case["past"]]
    rng = random.Random(case["past"] + case["batch"])
    return [rng.randint(case["past"] // 3, case["past"]) for _ in range(case["batch"])]


def _paths(case):
    """commit: a way from the root for each sequence, of a random length, [batch][nodes] padded
    with -1, and the lengths."""
    rng = random.Random(case["nodes"] + 3 * case["start"] + case["batch"])
    rows, trees = [], _trees(case)
    for b in range(case["batch"]):
        parents = trees[b % len(trees)]
        way, node = [], rng.randrange(case["nodes"])
        while node >= 0:
            way.append(node)
            node = parents[node]
        rows.append(way[::-1] + [-1] * (case["nodes"] - len(way)))
    return rows, [sum(n >= 0 for n in row) for row in rows]


def _ints(values, dtype=torch.int64):
    return torch.tensor(values, dtype=dtype, device="cuda") if values is not None else None


def _heads(gen, batch, seq, heads, head, std=1.0, dtype=torch.bfloat16):
    """[B, H, S, D] as the projections leave them: heads side by side in a row."""
    rows = torch.randn(batch, seq, heads, head, generator=gen, device="cuda") * std
    return rows.to(dtype).transpose(1, 2)


def _codes(gen, batch, heads, max_len, head):
    """Codes int8 [B, H, max_len, D] and scales [B, H, blocks] of a filled cache: the codes of
    normal values, 127 in each block's first token, scales of 8 significant bits (so that
    code x scale, and the largest of a block / 127, are exact in float32)."""
    blocks = -(-max_len // BLOCK)
    codes = torch.empty(batch, heads, max_len, head, dtype=torch.int8, device="cuda")
    for b in range(batch):
        x = torch.randn(heads, max_len, head, generator=gen, device="cuda") * 36.0
        codes[b] = x.round_().clamp_(-127, 127).to(torch.int8)
    codes[:, :, ::BLOCK, 0] = 127
    scales = (0.02 + 0.02 * torch.rand(batch, heads, blocks, generator=gen, device="cuda"))
    return codes, scales.to(torch.bfloat16).float()


def _values(codes, scales, dtype=torch.float32):
    """What codes [.., L, D] with scales [.., blocks] stand for."""
    per_token = scales.repeat_interleave(BLOCK, dim=-1)[..., :codes.shape[-2]]
    return codes.to(dtype) * per_token[..., None].to(dtype)


def _float_type(case):
    return torch.float32 if case["type"] == "f32" else torch.bfloat16


def _tree_inputs(case, gen):
    batch, heads, kv_heads, head, nodes, past = (
        case[n] for n in ("batch", "heads", "kv_heads", "head", "nodes", "past"))
    dtype = _float_type(case)
    x = {"q": _heads(gen, batch, nodes, heads, head, 1.5, dtype),
         "k": _heads(gen, batch, nodes, kv_heads, head, 1.0, dtype),
         "v": _heads(gen, batch, nodes, kv_heads, head, 1.0, dtype),
         "keys": _codes(gen, batch, kv_heads, past, head) if past else None,
         "values": _codes(gen, batch, kv_heads, past, head) if past else None,
         "start": _ints(_starts(case)), "parents": _ints(_trees(case), torch.int32),
         "counts": _ints(_counts(case)), "slopes": None}
    if case["slopes"]:  # falling geometrically over the heads
        powers = torch.arange(1, heads + 1, device="cuda", dtype=torch.float32) * (-8.0 / heads)
        x["slopes"] = torch.exp2(powers)
    return x


def _verify_inputs(case, gen):
    batch, nodes, vocab, dtype = case["batch"], case["nodes"], case["vocab"], _float_type(case)
    # four likely tokens and a long tail; the drafter's opinion is near the target's
    logits = torch.empty(batch, nodes, vocab, dtype=dtype, device="cuda")
    drafts = torch.empty_like(logits)
    children = torch.empty(batch, nodes, dtype=torch.int64, device="cuda")
    trees = _trees(case)
    for b in range(batch):
        base = torch.randn(nodes, vocab, generator=gen, device="cuda") * 1.5
        likely = torch.randint(vocab, (nodes, 4), generator=gen, device="cuda")
        more = torch.randn(nodes, 4, generator=gen, device="cuda") * 1.5
        base.scatter_(1, likely, more + math.log(vocab) + 2.0)
        logits[b] = base + torch.randn(nodes, vocab, generator=gen, device="cuda") * 0.5
        drafts[b] = base
        parents = _ints([max(p, 0) for p in trees[b % len(trees)]])
        # a node's token is drawn from the drafter's distribution at its parent
        scores = drafts[b][parents].float()
        if case["top_k"]:
            least = scores.topk(min(case["top_k"], vocab), dim=-1).values[:, -1:]
            scores = torch.where(scores < least, -math.inf, scores)
        noise = torch.rand(nodes, vocab, generator=gen, device="cuda").clamp_(min=1e-30)
        noise = -torch.log((-torch.log(noise)).clamp_(min=1e-30))
        children[b] = (scores + max(case["temperature"], 0.1) * noise).argmax(-1)
    x = {"logits": logits, "tokens": children, "drafts": drafts if case["drafter"] else None,
         "uniforms": torch.rand(batch, nodes, generator=gen, device="cuda"),
         "parents": _ints(trees, torch.int32), "counts": _ints(_counts(case))}
    return x


def _commit_inputs(case, gen):
    layers, batch, kv_heads, head, nodes = (case[n] for n in ("layers", "batch", "kv_heads",
                                                              "head", "nodes"))
    x = {n: [_heads(gen, batch, nodes, kv_heads, head) for _ in range(layers)] for n in "kv"}
    paths, counts = _paths(case)
    x.update(path=_ints(paths), counts=_ints(counts), start=_ints([case["start"]]))
    for name in ("keys", "values"):
        x[name] = None
        if case["start"]:
            x[name] = _codes(gen, layers * batch, kv_heads, case["start"], head)
    return x


def _inputs(case, seed):
    """The inputs alone, the same for either side."""
    gen = torch.Generator("cuda").manual_seed(seed)
    return {"tree": _tree_inputs, "verify": _verify_inputs,
            "commit": _commit_inputs}[case["kind"]](case, gen)


def _own():
    """The framework's modules (only where its kernels are measured)."""
    path = str(Path.cwd() / "local-ai-training_amd")
    if path not in sys.path:
        sys.path.insert(1, path)
    from local_ai_training import drafts, int8_cache

    return drafts, int8_cache


def _filled(x, batch, kv_heads, max_len, head):
    """The framework's cache with the codes of `x`, a sequence at a time (the values' float32 form
    is many times the cache)."""
    module = _own()[1]
    cache = module.int8_kv(batch, kv_heads, max_len, head, "cuda")
    begin = torch.zeros(1, dtype=torch.int64, device="cuda")
    for b in range(batch if x["keys"] is not None else 0):
        row = type(cache)(*(t[b:b + 1] for t in cache))
        module.int8_kv_append(row, _values(*(t[b:b + 1] for t in x["keys"])),
                              _values(*(t[b:b + 1] for t in x["values"])), begin)
    return cache


def prepare(case, seed):
    x = _inputs(case, seed)
    state = {"case": case, "x": x}
    kind = case["kind"]
    if own and kind != "commit":
        # a tree that all sequences share stays from step to step; others are planned in the pass
        state["tree"] = _own()[0].draft_tree(x["parents"]) if case["branch"] else None
    if kind == "tree":
        if own:
            # the program's cache has room for the nodes
            state["cache"] = _filled(x, case["batch"], case["kv_heads"],
                                     case["past"] + case["nodes"], case["head"])
            del x["keys"], x["values"]
        return state
    if kind == "verify":
        return state
    layers, batch, kv_heads, head = (case[n] for n in ("layers", "batch", "kv_heads", "head"))
    max_len = case["start"] + case["nodes"]
    if own:
        # the layers' caches side by side, in one allocation
        every = state["every"] = _filled(x, layers * batch, kv_heads, max_len, head)
        state["layers"] = [type(every)(*(t[i * batch:(i + 1) * batch] for t in every))
                           for i in range(layers)]
        del x["keys"], x["values"]
        return state
    for name in ("keys", "values"):
        codes = torch.zeros(layers * batch, kv_heads, max_len, head, dtype=torch.int8,
                            device="cuda")
        scales = torch.zeros(layers * batch, kv_heads, -(-max_len // BLOCK), device="cuda")
        if x[name] is not None:
            codes[:, :, :case["start"]] = x[name][0]
            scales[:, :, :x[name][1].shape[-1]] = x[name][1]
        state[name] = (codes, scales)
    return state


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"tree": _own_tree, "verify": _own_verify, "commit": _own_commit}[kind](state)
    return {"tree": _plain_tree, "verify": _plain_verify, "commit": _plain_commit}[kind](state)


def _own_tree(state):
    module = _own()[0]
    case, x = state["case"], state["x"]
    tree = state["tree"] or module.draft_tree(x["parents"])
    return [module.tree_attention(x["q"], x["k"], x["v"], state["cache"], x["start"], tree,
                                  lengths=x["counts"], softcap=case["cap"] or None,
                                  slopes=x["slopes"])]


def _own_verify(state):
    module = _own()[0]
    case, x = state["case"], state["x"]
    tree = state["tree"] or module.draft_tree(x["parents"])
    return list(module.verify_drafts(x["logits"], x["tokens"], tree, x["uniforms"],
                                     lengths=x["counts"], draft_logits=x["drafts"],
                                     temperature=case["temperature"],
                                     top_k=case["top_k"] or None))


def _touched(case):
    """The positions that a commit may write, from the first block's begin on."""
    longest = max(_paths(case)[1])
    return case["start"] // BLOCK * BLOCK, case["start"] + longest


def _own_commit(state):
    drafts, cache = _own()
    x = state["x"]
    drafts.int8_kv_commit(state["layers"], x["k"], x["v"], x["start"], x["path"], x["counts"])
    if "touched" not in state:
        state["touched"] = _touched(state["case"])
    return list(cache.int8_kv_read(state["every"], *state["touched"]))


def _lineage(parents):
    """Which node sees which, [rows, N, N], and the depths [rows, N], from the parents."""
    rows, nodes = parents.shape
    eye = torch.eye(nodes, device="cuda")
    step = torch.zeros(rows, nodes, nodes, device="cuda")
    if nodes > 1:
        step[:, 1:] = eye[parents[:, 1:].long()]
    seen, way = eye.expand(rows, nodes, nodes), step
    reach = 1
    while reach < nodes:  # ways of twice the length
        seen = ((seen + way @ seen) > 0).float()
        way = way @ way
        reach *= 2
    return seen > 0, seen.sum(-1) - 1.0


def _plain_tree(state):
    case, x = state["case"], state["x"]
    batch, heads, kv_heads, nodes, past = (case[n] for n in ("batch", "heads", "kv_heads", "nodes",
                                                             "past"))
    group, scale, cap = heads // kv_heads, 1.0 / math.sqrt(case["head"]), case["cap"]
    lineage, depths = _lineage(x["parents"])
    key_at = torch.arange(past, device="cuda")
    out = torch.empty(x["q"].shape, device="cuda")
    for b in range(batch):
        start = x["start"][b % x["start"].shape[0]]
        kin, depth = lineage[b % lineage.shape[0]], depths[b % depths.shape[0]]
        k, v = x["k"][b].float(), x["v"][b].float()
        if past:
            k = torch.cat([_values(*(t[b] for t in x["keys"])), k], dim=1)
            v = torch.cat([_values(*(t[b] for t in x["values"])), v], dim=1)
        q = x["q"][b].float().reshape(kv_heads, group * nodes, -1)
        s = (q @ k.transpose(1, 2).contiguous() * scale).view(heads, nodes, past + nodes)
        if cap:
            s = cap * torch.tanh(s / cap)
        if x["slopes"] is not None:
            distance = torch.cat([(start + depth)[:, None] - key_at[None, :],
                                  depth[:, None] - depth[None, :]], dim=1)
            s = s - x["slopes"][:, None, None] * distance
        seen = torch.cat([(key_at < start).expand(nodes, past), kin], dim=1)
        s = torch.where(seen, s, -math.inf)
        e = torch.exp(s - s.amax(-1, keepdim=True))
        p = (e / e.sum(-1, keepdim=True)).view(kv_heads, group * nodes, past + nodes)
        o = (p @ v).view(heads, nodes, -1)
        if x["counts"] is not None:
            there = torch.arange(nodes, device="cuda") < x["counts"][b]
            o = torch.where(there[None, :, None], o, 0.0)
        out[b] = o
    return [out.to(x["q"].dtype)]


def _distribution(logits, case):
    """The softmax of logits [.., V] over the temperature, in 64 bits, of the top_k largest."""
    x = logits.double() / case["temperature"]
    if case["top_k"]:
        least = logits.float().topk(min(case["top_k"], case["vocab"]), dim=-1).values[..., -1:]
        x = torch.where(logits.float() < least, -math.inf, x)
    e = torch.exp(x - x.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _plain_verify(state):
    case, x = state["case"], state["x"]
    batch, nodes, vocab = case["batch"], case["nodes"], case["vocab"]
    row = torch.arange(batch, device="cuda")
    parents = x["parents"].long().expand(batch, nodes)
    at = torch.zeros(batch, dtype=torch.int64, device="cuda")
    path = torch.full((batch, nodes), -1, dtype=torch.int64, device="cuda")
    path[:, 0] = 0
    count = torch.ones_like(at)
    greedy = case["temperature"] == 0.0
    if greedy:
        best = x["logits"].float().argmax(-1)
    else:
        p = _distribution(x["logits"], case)
        q = _distribution(x["drafts"], case) if x["drafts"] is not None else None
        left = p[:, 0]  # what is left of the distribution at the node
        total = torch.ones(batch, dtype=torch.float64, device="cuda")  # (its sum, no drafter)
    for i in range(1, nodes):
        tried = parents[:, i] == at
        if x["counts"] is not None:
            tried = tried & (i < x["counts"])
        token, u = x["tokens"][:, i], x["uniforms"][:, i].double()
        if greedy:
            stands = tried & (token == best[row, at])
        elif q is not None:
            stands = tried & (u * q[row, at, token] < left[row, token])
            rest = (left - q[row, at]).clamp(min=0.0)
            rest = rest / rest.sum(-1, keepdim=True)
        else:
            stands = tried & (u * total < left[row, token])
            rest = left.scatter(1, token[:, None], 0.0)
        if not greedy:
            left = torch.where(stands[:, None], p[:, i],
                               torch.where((tried & ~stands)[:, None], rest, left))
            if q is None:
                total = left.sum(-1)
        at = torch.where(stands, i, at)
        path[row, count.clamp(max=nodes - 1)] = torch.where(
            stands, i, path[row, count.clamp(max=nodes - 1)])
        count = count + stands
    if greedy:
        return [path, count, best[row, at]]
    sums = left.cumsum(-1)
    bound = x["uniforms"][:, 0].double() * sums[:, -1]
    token = (sums <= bound[:, None]).sum(-1).clamp(max=vocab - 1)
    return [path, count, token]


def _plain_commit(state):
    case, x = state["case"], state["x"]
    layers, batch, nodes = (case[n] for n in ("layers", "batch", "nodes"))
    (begin, end), start = _touched(case), case["start"]
    longest, outputs = end - start, []
    most = torch.tensor(127.0, device="cuda")
    way = x["path"].clamp(min=0)[:, :longest]
    there = (torch.arange(longest, device="cuda") < x["counts"][:, None]).repeat(layers, 1)
    row = torch.arange(batch, device="cuda")[:, None]
    for name, given in (("keys", x["k"]), ("values", x["v"])):
        codes, scales = state[name]
        new = torch.cat([t.transpose(1, 2)[row, way].transpose(1, 2) for t in given]).float()
        new = torch.where(there[:, None, :, None], new, 0.0)
        for low in range(begin, end, BLOCK):
            high, block = min(low + BLOCK, end), low // BLOCK
            kept = max(low, start)
            part = new[:, :, kept - start:high - start]
            some = there[:, kept - start:high - start]
            old = scales[:, :, block]
            s = part.abs().amax((2, 3)) / most
            if kept > low:
                s = torch.maximum(s, old)
                ratio = (old / torch.where(s > 0, s, 1.0))[:, :, None, None]
                codes[:, :, low:kept] = (codes[:, :, low:kept].float() * ratio).round().to(torch.int8)
            # a block that a sequence does not reach stays as it is
            s = torch.where(some.any(1)[:, None], s, old)
            scales[:, :, block] = s
            rows = (part / torch.where(s > 0, s, 1.0)[:, :, None, None]).round()
            codes[:, :, kept:high] = torch.where(some[:, None, :, None], rows.to(torch.int8),
                                                 codes[:, :, kept:high])
        outputs.append(_values(codes[:, :, begin:end], scales[:, :, begin // BLOCK:]))
    return outputs


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    x = _inputs(case, seed)
    return {"tree": _exact_tree, "verify": _exact_verify, "commit": _exact_commit}[case["kind"]](
        case, x)


def _exact_tree(case, x):
    nodes, group = case["nodes"], case["heads"] // case["kv_heads"]
    starts, trees, counts = _starts(case), _trees(case), _counts(case)
    slopes = x["slopes"].double() if x["slopes"] is not None else None
    out = torch.zeros(x["q"].shape, dtype=torch.float64, device="cuda")
    for b in range(case["batch"]):
        start, parents = starts[b % len(starts)], trees[b % len(trees)]
        there = counts[b] if counts else nodes
        depths = _depths(parents)
        seen = torch.zeros(there, start + nodes, dtype=torch.bool)
        seen[:, :start] = True
        for i in range(there):
            node = i
            while node >= 0:
                seen[i, start + node] = True
                node = parents[node]
        seen = seen.cuda()
        at = _ints(list(range(start)) + [start + d for d in depths]).double()
        distance = at[start:start + there, None] - at[None, :]
        for kv in range(case["kv_heads"]):
            k, v = x["k"][b, kv].double(), x["v"][b, kv].double()
            if start:
                k, v = (torch.cat([_values(x[n][0][b, kv, :start], x[n][1][b, kv], torch.float64),
                                   t]) for n, t in (("keys", k), ("values", v)))
            for h in range(kv * group, (kv + 1) * group):
                s = torch.mm(x["q"][b, h, :there].double(), k.t()) / math.sqrt(case["head"])
                if case["cap"]:
                    s = case["cap"] * torch.tanh(s / case["cap"])
                if slopes is not None:
                    s = s - slopes[h] * distance
                out[b, h, :there] = torch.mm(torch.softmax(s.masked_fill(~seen, -math.inf), 1), v)
    return [out]


def _exact_row(logits, case):
    z = logits.double()
    if case["top_k"]:
        order = torch.sort(z, descending=True).values
        z = z.masked_fill(z < order[min(case["top_k"], case["vocab"]) - 1], -math.inf)
    return torch.softmax(z / case["temperature"], 0)


def _exact_verify(case, x):
    trees, counts = _trees(case), _counts(case)
    tokens, uniforms = x["tokens"].tolist(), x["uniforms"].double().tolist()
    paths, lengths, following = [], [], []
    for b in range(case["batch"]):
        parents = trees[b % len(trees)]
        there = counts[b] if counts else case["nodes"]
        way, follow = [0], None
        while follow is None:
            node = way[-1]
            children = [i for i in range(there) if parents[i] == node]
            row = x["logits"][b, node]
            if case["temperature"] == 0.0:
                follow = int(torch.nonzero(row == row.max())[0])
                way += [i for i in children if tokens[b][i] == follow][:1]
            else:
                p = _exact_row(row, case)
                q = None
                if children and x["drafts"] is not None:
                    q = _exact_row(x["drafts"][b, node], case)
                for i in children:
                    token = tokens[b][i]
                    chance = 1.0 if q is None else float(q[token])
                    if uniforms[b][i] * chance < float(p[token]):
                        way.append(i)
                        break
                    if q is None:
                        p = p.clone()
                        p[token] = 0.0
                    else:
                        p = torch.relu(p - q)
                    p = p / p.sum()
                if way[-1] == node:
                    sums = torch.cumsum(p, 0)
                    bound = uniforms[b][0] * float(sums[-1])
                    follow = int(torch.nonzero(sums > bound)[0])
            if way[-1] != node:
                follow = None
        paths.append(way + [-1] * (case["nodes"] - len(way)))
        lengths.append(len(way))
        following.append(follow)
    return [_ints(paths), _ints(lengths), _ints(following)]


def _f32(x):
    """Rounded to a float32 number, held in 64 bits."""
    return x.float().double()


def _exact_commit(case, x):
    batch, start = case["batch"], case["start"]
    begin, end = _touched(case)
    paths, counts = _paths(case)
    outputs = []
    for name, given in (("keys", x["k"]), ("values", x["v"])):
        out = torch.zeros(case["layers"] * batch, case["kv_heads"], end - begin, case["head"],
                          dtype=torch.float64, device="cuda")
        for i in range(case["layers"] * batch):
            layer, b = divmod(i, batch)
            fresh = given[layer][b][:, paths[b][:counts[b]]].double()
            for low in range(begin, start + counts[b], BLOCK):
                kept, high = max(low, start), min(low + BLOCK, start + counts[b])
                part = fresh[:, kept - start:high - start]
                s = _f32(part.abs().flatten(1).amax(1)[:, None, None] / 127.0)
                if kept > low:
                    codes, scales = x[name]
                    old = scales[i, :, low // BLOCK].double()[:, None, None]
                    s = torch.maximum(s, old)
                    again = torch.round(_f32(codes[i, :, low:kept].double() * _f32(old / s)))
                    out[i, :, low - begin:kept - begin] = again * s
                out[i, :, kept - begin:high - begin] = torch.round(_f32(part / s)) * s
        outputs.append(out)
    return outputs


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    kind, batch, nodes = case["kind"], case["batch"], case["nodes"]
    if kind == "tree":
        heads, kv_heads, head = case["heads"], case["kv_heads"], case["head"]
        starts, trees, counts = _starts(case), _trees(case), _counts(case)
        tokens = pairs = 0
        for b in range(batch):
            there = counts[b] if counts else nodes
            depths = _depths(trees[b % len(trees)])[:there]
            tokens += starts[b % len(starts)]
            pairs += there * starts[b % len(starts)] + sum(d + 1 for d in depths)
        size = 4.0 if case["type"] == "f32" else 2.0
        # codes and scales, k and v of the nodes; q in, the result out
        nbytes = 2.0 * kv_heads * (tokens * head + 4.0 * tokens / BLOCK) \
            + 2.0 * size * batch * nodes * head * (heads + kv_heads)
        return {"bytes": nbytes, "flops": 4.0 * head * pairs * heads}
    if kind == "verify":
        size = 4.0 if case["type"] == "f32" else 2.0
        trees, counts = _trees(case), _counts(case)
        rows = 0
        for b in range(batch):
            there = counts[b] if counts else nodes
            rows += there
            if case["drafter"] and case["temperature"]:  # where a node has children
                rows += len({p for p in trees[b % len(trees)][:there] if p >= 0})
        # a comparison for the largest, an exponential and a sum a logit
        return {"bytes": size * rows * case["vocab"] + 24.0 * batch * nodes,
                "flops": 3.0 * rows * case["vocab"]}
    counts = _paths(case)[1]
    begin, end = _touched(case)
    # the nodes' rows in (2 bytes) and their codes out, the touched tokens read back as float32
    per_head = sum(n * (2 + 1) + (end - begin) * (1 + 4) for n in counts)
    values = 2.0 * case["layers"] * case["kv_heads"] * case["head"]
    return {"bytes": values * per_head, "flops": values * (3 * sum(counts) + batch * (end - begin))}
