"""Attention with modified scores, and the 8-bit key/value cache it is served from: what a
program that trains on packed documents and then generates has these operators do.

Kinds of case:

* ``scored``: attention whose scores are capped by a tanh, get a bias that falls with the
  distance, and are masked by documents and by the marked prefix of each document; the mask's
  plan is made within the pass. With ``train`` the gradients of q, k, v (and of the slopes, where
  there are any) come with the output.
* ``append``: keys and values written into a cache of 8-bit codes with one scale per block of 64
  tokens and head, and the touched blocks read back.
* ``read``: attention of one or more new tokens per sequence over such a cache.

Head counts and sizes are those of the 25M (8 heads of 64, window 512) and the 1B transformer
(16 heads of 128, window 1024) that the benchmark and the tests run, or generic.

Definitions. A document is a run of equal ids >= 0; negative ids are padding, which sees nothing
and is seen by nothing. Query i sees key j of its document if j <= i or if j lies in the run of
marked positions that the document begins with. The score is scale q.k, then cap tanh(. / cap),
then minus slope_h |i - j|. A row that sees nothing gives zeros.

A cache block's scale is its largest absolute value / 127 and a code is rint(x / scale). Appended
tokens can only raise the scale s of a block that already holds tokens: to
max(s, largest new value / 127); its codes c are then rounded again, rint(c (s / s_new)). Scales,
quotients and ratios are float32 numbers, as in the framework's row quantization, so the codes
are defined to the last one.
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
        # a small batch of short rows with prompts that see themselves whole: latency counts
        {"name": "scored_tiny", "kind": "scored", "batch": 2, "heads": 4, "kv_heads": 4,
         "seq": 37, "head": 64, "cap": 0.0, "slopes": False, "doc": 0, "prefix": True,
         "pad": False, "train": True},
        # the 25M model's attention layer on packed documents
        {"name": "scored_packed_25m", "kind": "scored", "batch": 32, "heads": 8, "kv_heads": 8,
         "seq": 512, "head": 64, "cap": 0.0, "slopes": False, "doc": 150, "prefix": False,
         "pad": False, "train": True},
        # the 1B model's attention layer with capped scores, packed documents
        {"name": "scored_capped_1b", "kind": "scored", "batch": 8, "heads": 16, "kv_heads": 16,
         "seq": 1024, "head": 128, "cap": 30.0, "slopes": False, "doc": 400, "prefix": False,
         "pad": False, "train": True},
        # the 1B model's attention layer with a distance bias that is learned, no documents, an
        # odd length
        {"name": "scored_bias_1b", "kind": "scored", "batch": 4, "heads": 16, "kv_heads": 16,
         "seq": 1001, "head": 128, "cap": 0.0, "slopes": True, "doc": 0, "prefix": False,
         "pad": False, "train": True},
        # one long packed row with shared key heads and everything switched on
        {"name": "scored_long_shared", "kind": "scored", "batch": 1, "heads": 16, "kv_heads": 4,
         "seq": 8192, "head": 128, "cap": 50.0, "slopes": True, "doc": 4000, "prefix": True,
         "pad": False, "train": True},
        # prompts of several lengths in one padded batch, forward only
        {"name": "scored_prompts", "kind": "scored", "batch": 16, "heads": 16, "kv_heads": 16,
         "seq": 777, "head": 128, "cap": 0.0, "slopes": False, "doc": 0, "prefix": True,
         "pad": True, "train": False},
        # prompts of the 1B model into an empty cache
        {"name": "append_prompt", "kind": "append", "batch": 4, "kv_heads": 16, "head": 128,
         "start": 0, "new": 777, "max_len": 1024},
        # one generated token per sequence into blocks that already hold some
        {"name": "append_token", "kind": "append", "batch": 16, "kv_heads": 16, "head": 128,
         "start": 965, "new": 1, "max_len": 1024},
        # generation with the 1B model, one sequence
        {"name": "read_b1", "kind": "read", "batch": 1, "heads": 16, "kv_heads": 16, "head": 128,
         "past": 1000, "ragged": False, "new": 1, "max_len": 1024, "cap": 0.0, "slopes": False},
        # generation for a batch of long sequences of several lengths, with a distance bias
        {"name": "read_b16_long", "kind": "read", "batch": 16, "heads": 16, "kv_heads": 16,
         "head": 128, "past": 16000, "ragged": True, "new": 1, "max_len": 16384, "cap": 0.0,
         "slopes": True},
        # generation for many sequences with shared key heads and capped scores
        {"name": "read_shared_b48", "kind": "read", "batch": 48, "heads": 32, "kv_heads": 4,
         "head": 64, "past": 8100, "ragged": True, "new": 1, "max_len": 8192, "cap": 30.0,
         "slopes": False},
        # the next part of long prompts over what the cache holds of them
        {"name": "read_chunk", "kind": "read", "batch": 4, "heads": 16, "kv_heads": 16,
         "head": 128, "past": 1500, "ragged": False, "new": 517, "max_len": 2048, "cap": 0.0,
         "slopes": True},
    ]


def _between(rng, low, high):
    """An integer spread over the logarithm of its range."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["scored", "scored", "append", "read", "read"])
    head = rng.choice([64, 128])
    if kind == "scored":
        heads = rng.choice([1, 4, 6, 8, 12, 16])
        kv_heads = heads // rng.choice([g for g in (1, 1, 2, 4) if heads % g == 0])
        seq = _between(rng, 1, 8192)
        most = max(1, min(32, int(16 * 8192.0**2 / (heads * max(seq, 64)**2))))
        batch = _between(rng, 1, most)
        doc = rng.choice([0, _between(rng, 1, seq)])
        return {"kind": kind, "batch": batch, "heads": heads, "kv_heads": kv_heads, "seq": seq,
                "head": head, "cap": rng.choice([0.0, rng.uniform(5.0, 50.0)]),
                "slopes": rng.random() < 0.5, "doc": doc, "prefix": rng.random() < 0.5,
                "pad": rng.random() < 0.3, "train": rng.random() < 0.7}
    batch = _between(rng, 1, 48)
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    if kind == "append":
        new = rng.choice([1, _between(rng, 2, 1500)])
        start = rng.randint(0, 900)
        return {"kind": kind, "batch": min(batch, 16), "kv_heads": kv_heads, "head": head,
                "start": start, "new": new, "max_len": start + new + rng.randint(0, 200)}
    heads = kv_heads * rng.choice([1, 1, 2, 4, 8])
    new = rng.choice([1, 1, _between(rng, 2, 600)])
    # the cache of the largest listed case: 16 x 16 x 16384 x 128 codes
    longest = max(64, min(16000, 16 * 16 * 16384 // (batch * max(heads, 1)) // (1 + new // 32)))
    past = _between(rng, 1, longest)
    return {"kind": kind, "batch": batch, "heads": heads, "kv_heads": kv_heads, "head": head,
            "past": past, "ragged": rng.random() < 0.5, "new": new,
            "max_len": past + new + rng.randint(0, 100),
            "cap": rng.choice([0.0, rng.uniform(5.0, 50.0)]), "slopes": rng.random() < 0.5}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _documents(case):
    """Document ids [B][S] of a case (its own, whatever the seed): lengths spread about the mean,
    every one at least one token; padded cases end in up to half a row of padding."""
    rng = random.Random(1009 * case["seq"] + 31 * case["batch"] + case["doc"])
    rows = []
    for b in range(case["batch"]):
        ids, number = [], 0
        while len(ids) < case["seq"]:
            length = case["seq"]
            if case["doc"]:
                length = max(1, round(case["doc"] * rng.uniform(0.25, 1.75)))
            ids += [number] * length
            number += 1
        ids = ids[:case["seq"]]
        if case["pad"]:
            kept = rng.randint(case["seq"] // 2, case["seq"])
            ids = ids[:kept] + [-1] * (case["seq"] - kept)
        rows.append(ids)
    return rows


def _marks(case, rows):
    """Marked positions [B][S]: each document begins with a marked run (its prompt)."""
    rng = random.Random(7 * case["seq"] + case["batch"])
    marks = []
    for ids in rows:
        row, left = [], 0
        for i, number in enumerate(ids):
            if i == 0 or number != ids[i - 1]:
                left = rng.randint(0, 1 + (case["doc"] or case["seq"]) // 2)
            row.append(left > 0)
            left -= 1
        marks.append(row)
    return marks


def _slopes(heads, gen, learned):
    """Slopes falling geometrically over the heads; learned ones have moved a little."""
    powers = torch.arange(1, heads + 1, device="cuda", dtype=torch.float32) * (-8.0 / heads)
    noise = 1.0 + 0.1 * torch.randn(heads, generator=gen, device="cuda")
    return (torch.exp2(powers) * noise).requires_grad_(learned)


def _heads(gen, batch, seq, heads, head, std=1.0):
    """bf16 [B, H, S, D] as the projections leave them: heads side by side in a row."""
    rows = torch.randn(batch, seq, heads, head, generator=gen, device="cuda") * std
    return rows.to(torch.bfloat16).transpose(1, 2)


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


def _inputs(case, seed):
    """The inputs alone, the same for either side."""
    gen = torch.Generator("cuda").manual_seed(seed)
    kind, batch, head = case["kind"], case["batch"], case["head"]
    if kind == "scored":
        seq, heads, kv_heads = case["seq"], case["heads"], case["kv_heads"]
        x = {"q": _heads(gen, batch, seq, heads, head), "k": _heads(gen, batch, seq, kv_heads, head),
             "v": _heads(gen, batch, seq, kv_heads, head)}
        x["slopes"] = _slopes(heads, gen, case["train"]) if case["slopes"] else None
        rows = _documents(case)
        masked = case["doc"] or case["pad"]
        x["documents"] = torch.tensor(rows, device="cuda") if masked else None
        x["prefix"] = torch.tensor(_marks(case, rows), device="cuda") if case["prefix"] else None
        if case["train"]:
            for name in ("q", "k", "v"):
                x[name] = x[name].requires_grad_()
            x["grad"] = _heads(gen, batch, seq, heads, head)
        return x
    kv_heads, max_len = case["kv_heads"], case["max_len"]
    if kind == "append":
        x = {"start": torch.tensor([case["start"]], device="cuda"),
             "k": _heads(gen, batch, case["new"], kv_heads, head),
             "v": _heads(gen, batch, case["new"], kv_heads, head)}
        x["keys"] = _codes(gen, batch, kv_heads, case["start"], head) if case["start"] else None
        x["values"] = _codes(gen, batch, kv_heads, case["start"], head) if case["start"] else None
        return x
    filled = case["past"] + case["new"]
    x = {"q": _heads(gen, batch, case["new"], case["heads"], head, 1.5),
         "keys": _codes(gen, batch, kv_heads, filled, head),
         "values": _codes(gen, batch, kv_heads, filled, head),
         "slopes": _slopes(case["heads"], gen, False) if case["slopes"] else None}
    start = torch.full((batch,), case["past"], dtype=torch.int64)
    if case["ragged"]:
        rng = random.Random(case["past"] + batch)
        start = torch.tensor([rng.randint(case["past"] // 3, case["past"]) for _ in range(batch)])
    x["start"] = start.cuda() if case["ragged"] else start[:1].cuda()
    return x


def _own():
    """The framework's modules (only where its kernels are measured)."""
    path = str(Path.cwd() / "local-ai-training_amd")
    if path not in sys.path:
        sys.path.insert(1, path)
    from local_ai_training import int8_cache, scored_attention

    return scored_attention, int8_cache


def prepare(case, seed):
    x = _inputs(case, seed)
    state = {"case": case, "x": x}
    if case["kind"] == "scored":
        return state
    batch, kv_heads, head, max_len = (case[n] for n in ("batch", "kv_heads", "head", "max_len"))
    if own:
        cache_module = _own()[1]
        cache = cache_module.int8_kv(batch, kv_heads, max_len, head, x["q" if "q" in x else "k"].device)
        if x["keys"] is not None:
            begin = torch.zeros(1, dtype=torch.int64, device="cuda")
            # a sequence at a time: the values' float32 form is many times the cache
            for b in range(batch):
                row = type(cache)(*(t[b:b + 1] for t in cache))
                cache_module.int8_kv_append(row, _values(*(t[b:b + 1] for t in x["keys"])),
                                            _values(*(t[b:b + 1] for t in x["values"])), begin)
        state["cache"] = cache
        if case["kind"] == "read":
            del x["keys"], x["values"]
        return state
    if case["kind"] == "append":
        blocks = -(-max_len // BLOCK)
        for name in ("keys", "values"):
            codes = torch.zeros(batch, kv_heads, max_len, head, dtype=torch.int8, device="cuda")
            scales = torch.zeros(batch, kv_heads, blocks, device="cuda")
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
        return {"scored": _own_scored, "append": _own_append, "read": _own_read}[kind](state)
    return {"scored": _plain_scored, "append": _plain_append, "read": _plain_read}[kind](state)


def _own_scored(state):
    module = _own()[0]
    case, x = state["case"], state["x"]
    mask = None
    if x["documents"] is not None or x["prefix"] is not None:
        mask = module.attention_mask(documents=x["documents"], prefix=x["prefix"])
    out = module.scored_attention(x["q"], x["k"], x["v"], mask=mask, softcap=case["cap"] or None,
                                  slopes=x["slopes"])
    if not case["train"]:
        return [out]
    leaves = [x["q"], x["k"], x["v"]] + ([x["slopes"]] if case["slopes"] else [])
    return [out.detach(), *torch.autograd.grad(out, leaves, x["grad"])]


def _touched(case):
    return case["start"] // BLOCK * BLOCK, case["start"] + case["new"]


def _own_append(state):
    module, x = _own()[1], state["x"]
    module.int8_kv_append(state["cache"], x["k"], x["v"], x["start"])
    return list(module.int8_kv_read(state["cache"], *_touched(state["case"])))


def _own_read(state):
    case, x = state["case"], state["x"]
    return [_own()[1].int8_kv_attention(x["q"], state["cache"], x["start"],
                                        softcap=case["cap"] or None, slopes=x["slopes"])]


def _seen(documents, prefix, batch, seq):
    """Which key each query sees, [B, S, S]."""
    at = torch.arange(seq, device="cuda")
    if documents is None:
        documents = torch.zeros(batch, seq, dtype=torch.int64, device="cuda")
    first = torch.ones_like(documents, dtype=torch.bool)
    first[:, 1:] = documents[:, 1:] != documents[:, :-1]
    number = first.cumsum(1)
    real = documents >= 0
    seen = (number[:, :, None] == number[:, None, :]) & real[:, :, None] & real[:, None, :]
    earlier = at[None, :] <= at[:, None]
    if prefix is None:
        return seen & earlier
    # the last unmarked position up to each one; the run is unbroken if its document begins later
    broken = torch.where(prefix, -1, at).cummax(1).values
    begin = torch.where(first, at, 0).cummax(1).values
    return seen & (earlier | (broken < begin)[:, None, :])


def _weights(scores, cap, slopes, seen, distance):
    """Softmax of the modified scores [N, Q, K]; also tanh's value, for the gradient."""
    t = torch.tanh(scores / cap) if cap else None
    scores = cap * t if cap else scores
    if slopes is not None:
        scores = scores - slopes[:, None, None] * distance
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, 1.0, total), t


def _plain_scored(state):
    case, x = state["case"], state["x"]
    batch, heads, kv_heads, seq, head = (case[n] for n in ("batch", "heads", "kv_heads", "seq",
                                                           "head"))
    group, scale, cap = heads // kv_heads, 1.0 / math.sqrt(head), case["cap"]
    at = torch.arange(seq, device="cuda")
    distance = (at[:, None] - at[None, :]).abs().float() if case["slopes"] else None
    q, k, v = (x[n].detach().float() for n in ("q", "k", "v"))
    out = torch.empty(batch, heads, seq, head, device="cuda")
    dq, dk, dv = torch.empty_like(out), torch.zeros_like(k), torch.zeros_like(v)
    dslopes = torch.zeros(heads, dtype=torch.float64, device="cuda")
    every = _seen(x["documents"], x["prefix"], batch, seq)
    step = max(1, min(heads, (1 << 27) // (seq * seq)))
    for b in range(batch):
        for h in range(0, heads, step):
            hs = slice(h, min(h + step, heads))
            kv = torch.arange(hs.start, hs.stop, device="cuda") // group
            qs, ks, vs = q[b, hs].contiguous(), k[b, kv].contiguous(), v[b, kv].contiguous()
            slopes = x["slopes"].detach()[hs] if case["slopes"] else None
            p, t = _weights(qs @ ks.transpose(1, 2).contiguous() * scale, cap, slopes, every[b],
                            distance)
            o = p @ vs
            out[b, hs] = o
            if not case["train"]:
                continue
            g = x["grad"][b, hs].float().contiguous()
            dv[b].index_add_(0, kv, p.transpose(1, 2).contiguous() @ g)
            ds = p * (g @ vs.transpose(1, 2).contiguous() - (g * o).sum(-1, keepdim=True))
            if slopes is not None:
                dslopes[hs] -= (ds * distance).sum(-1).double().sum(-1)
            if cap:
                ds = ds * (1.0 - t * t)
            ds = ds * scale
            dq[b, hs] = ds @ ks
            dk[b].index_add_(0, kv, ds.transpose(1, 2).contiguous() @ qs)
    outputs = [out, dq, dk, dv] if case["train"] else [out]
    outputs = [t.to(torch.bfloat16) for t in outputs]
    return outputs + [dslopes.float()] if case["train"] and case["slopes"] else outputs


def _plain_append(state):
    case, x = state["case"], state["x"]
    begin, end = _touched(case)
    start, outputs = case["start"], []
    most = torch.tensor(127.0, device="cuda")
    for name, new in (("keys", x["k"].float()), ("values", x["v"].float())):
        codes, scales = state[name]
        for low in range(begin, end, BLOCK):
            high, block = min(low + BLOCK, end), low // BLOCK
            kept = max(low, start)
            part = new[:, :, kept - start:high - start]
            s = part.abs().amax((2, 3)) / most
            if kept > low:
                s = torch.maximum(s, scales[:, :, block])
                ratio = (scales[:, :, block] / torch.where(s > 0, s, 1.0))[:, :, None, None]
                codes[:, :, low:kept] = (codes[:, :, low:kept].float() * ratio).round().to(torch.int8)
            scales[:, :, block] = s
            rows = (part / torch.where(s > 0, s, 1.0)[:, :, None, None]).round()
            codes[:, :, kept:high] = rows.to(torch.int8)
        outputs.append(_values(codes[:, :, begin:end], scales[:, :, begin // BLOCK:]))
    return outputs


def _plain_read(state):
    case, x = state["case"], state["x"]
    batch, heads, kv_heads, new, head = (case[n] for n in ("batch", "heads", "kv_heads", "new",
                                                           "head"))
    group, scale = heads // kv_heads, 1.0 / math.sqrt(head)
    total = case["past"] + new
    key_at = torch.arange(total, device="cuda")
    out = torch.empty(batch, heads, new, head, device="cuda")
    for b in range(batch):
        at = x["start"][b if case["ragged"] else 0] + torch.arange(new, device="cuda")
        distance = (at[:, None] - key_at[None, :]).abs().float()
        seen = key_at[None, :] <= at[:, None]
        k, v = _values(*(t[b] for t in x["keys"])), _values(*(t[b] for t in x["values"]))
        k, v = (t.repeat_interleave(group, dim=0) for t in (k, v))
        q = x["q"][b].float().contiguous()
        p, _ = _weights(q @ k.transpose(1, 2).contiguous() * scale, case["cap"], x["slopes"],
                        seen, distance)
        out[b] = p @ v
    return [out.to(torch.bfloat16)]


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    x = _inputs(case, seed)
    return {"scored": _exact_scored, "append": _exact_append, "read": _exact_read}[case["kind"]](
        case, x)


def _exact_row(q, k, v, seen, distance, cap, slope):
    """One head: q [Q, D], k, v [K, D] float64; -> [Q, D]."""
    s = torch.mm(q, k.t()) / math.sqrt(q.shape[1])
    if cap:
        s = cap * torch.tanh(s / cap)
    if slope is not None:
        s = s - slope * distance
    s = s.masked_fill(~seen, -math.inf)
    empty = ~seen.any(1, keepdim=True)
    return torch.mm(torch.softmax(s.masked_fill(empty, 0.0), 1).masked_fill(empty, 0.0), v)


def _exact_seen(case, b):
    """[S, S] of row b, from the case's documents one at a time."""
    rows = _documents(case)
    marks = _marks(case, rows)[b] if case["prefix"] else None
    ids, seq = rows[b], case["seq"]
    seen = torch.zeros(seq, seq, dtype=torch.bool, device="cuda")
    low = 0
    while low < seq:
        high = low
        while high < seq and ids[high] == ids[low]:
            high += 1
        if ids[low] >= 0:
            part = torch.ones(high - low, high - low, dtype=torch.bool, device="cuda").tril()
            lead = 0
            while marks is not None and low + lead < high and marks[low + lead]:
                lead += 1
            part[:, :lead] = True
            seen[low:high, low:high] = part
        low = high
    return seen


def _exact_scored(case, x):
    batch, heads, seq = case["batch"], case["heads"], case["seq"]
    group, train = heads // case["kv_heads"], case["train"]
    at = torch.arange(seq, device="cuda", dtype=torch.float64)
    distance = (at[:, None] - at[None, :]).abs() if case["slopes"] else None
    slopes = x["slopes"].detach().double() if case["slopes"] else None
    out = torch.empty(x["q"].shape, dtype=torch.float64, device="cuda")
    grads = [torch.zeros(x[n].shape, dtype=torch.float64, device="cuda") for n in ("q", "k", "v")]
    dslopes = torch.zeros(heads, dtype=torch.float64, device="cuda")
    for b in range(batch):
        seen = _exact_seen(case, b)
        for h in range(heads):
            leaves = [t.detach()[b, i].double().requires_grad_(train)
                      for t, i in ((x["q"], h), (x["k"], h // group), (x["v"], h // group))]
            slope = slopes[h].clone().requires_grad_(train) if slopes is not None else None
            o = _exact_row(*leaves, seen, distance, case["cap"], slope)
            out[b, h] = o.detach()
            if train:
                wanted = leaves + ([slope] if slope is not None else [])
                got = torch.autograd.grad(o, wanted, x["grad"][b, h].double())
                grads[0][b, h] = got[0]
                grads[1][b, h // group] += got[1]
                grads[2][b, h // group] += got[2]
                if slope is not None:
                    dslopes[h] += got[3]
    if not train:
        return [out]
    return [out, *grads] + ([dslopes] if slopes is not None else [])


def _f32(x):
    """Rounded to a float32 number, held in 64 bits."""
    return x.float().double()


def _exact_append(case, x):
    begin, end = _touched(case)
    start, outputs = case["start"], []
    for name, new in (("keys", x["k"].double()), ("values", x["v"].double())):
        parts = []
        for low in range(begin, end, BLOCK):
            high, kept = min(low + BLOCK, end), max(low, start)
            fresh = new[:, :, kept - start:high - start]
            s = _f32(fresh.abs().flatten(2).amax(2)[:, :, None, None] / 127.0)
            if kept > low:
                codes, scales = x[name]
                old = scales[:, :, low // BLOCK].double()[:, :, None, None]
                s = torch.maximum(s, old)
                again = codes[:, :, low:kept].double() * _f32(old / s)
                parts.append(torch.round(_f32(again)) * s)
            parts.append(torch.round(_f32(fresh / s)) * s)
        outputs.append(torch.cat(parts, 2))
    return outputs


def _exact_read(case, x):
    batch, heads, new = case["batch"], case["heads"], case["new"]
    group = heads // case["kv_heads"]
    slopes = x["slopes"].double() if case["slopes"] else None
    out = torch.empty(batch, heads, new, case["head"], dtype=torch.float64, device="cuda")
    starts = x["start"].tolist()
    for b in range(batch):
        start = starts[b % len(starts)]
        keys = torch.arange(start + new, device="cuda")
        at = start + torch.arange(new, device="cuda")
        distance = (at[:, None] - keys[None, :]).double().abs()
        for kv in range(case["kv_heads"]):
            k, v = (_values(x[n][0][b, kv], x[n][1][b, kv], torch.float64)[:start + new]
                    for n in ("keys", "values"))
            for h in range(kv * group, (kv + 1) * group):
                out[b, h] = _exact_row(x["q"][b, h].double(), k, v, _up_to(at, keys),
                                       distance, case["cap"],
                                       slopes[h] if slopes is not None else None)
    return [out]


def _up_to(at, keys):
    """A query at position `at` sees the keys up to it."""
    return keys[None, :] <= at[:, None]


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    batch, head = case["batch"], case["head"]
    kv_heads = case["kv_heads"]
    if case["kind"] == "scored":
        heads, seq, train = case["heads"], case["seq"], case["train"]
        rows = _documents(case)
        marks = _marks(case, rows) if case["prefix"] else None
        pairs = 0
        for b, ids in enumerate(rows):
            low = 0
            while low < seq:
                high = low
                while high < seq and ids[high] == ids[low]:
                    high += 1
                lead = 0
                while marks is not None and low + lead < high and marks[b][low + lead]:
                    lead += 1
                if ids[low] >= 0:
                    n = high - low
                    pairs += n * (n + 1) // 2 + lead * (lead - 1) // 2
                low = high
        # two products forward, five backward, 2 D operations a pair each
        flops = 2.0 * head * pairs * heads * (7 if train else 2)
        # q, o and k, v; with gradients also do, dq and dk, dv
        nbytes = 2.0 * batch * seq * head * ((4 if train else 2) * heads
                                             + (4 if train else 2) * kv_heads)
        return {"bytes": nbytes, "flops": flops}
    if case["kind"] == "append":
        begin, end = _touched(case)
        new = case["new"]
        # new rows in (2 bytes) and their codes out, the touched tokens read back as float32
        per_head = new * (2 + 1) + (end - begin) * (1 + 4)
        return {"bytes": 2.0 * batch * kv_heads * head * per_head,
                "flops": 2.0 * batch * kv_heads * head * (3 * new + end - begin)}
    new, heads = case["new"], case["heads"]
    past = case["past"]
    if case["ragged"]:
        rng = random.Random(past + batch)
        starts = [rng.randint(past // 3, past) for _ in range(batch)]
    else:
        starts = [past] * batch
    tokens = sum(s + new for s in starts)
    pairs = sum(new * s + new * (new + 1) // 2 for s in starts)
    nbytes = 2.0 * kv_heads * (tokens * head + 4.0 * tokens / BLOCK) \
        + 4.0 * batch * heads * new * head
    return {"bytes": nbytes, "flops": 4.0 * head * pairs * heads}
