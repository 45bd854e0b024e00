"""Operators for several continuations of one prompt, as cases to time: attention of queries that share the cached rows of
a prompt, and copies of cached rows between the sequences of a cache (forks, reorderings, compactions).

A case is a dict of plain values; all lengths follow from it alone.  ``prepare`` makes what a program holds before the call,
``run`` is one call of the framework's operator, or its plain form in 32 bits where ``own`` is false.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed() -> list[dict]:
    return [
        # two samples of a small puzzle with the smallest grid model: a step of an interactive caller
        dict(name="two samples, one puzzle", kind="attend", heads=4, kv=4, dim=64, act="f16", cache="bf16", groups=1, items=2, prefix=190, own=17),
        # sixteen samples of the longest puzzle (five pairs of 30 x 30 grids) with the large grid model
        dict(name="sixteen samples, long puzzle", kind="attend", heads=20, kv=20, dim=64, act="f16", cache="bf16", groups=1, items=16, prefix=10247, own=931),
        # the augmentation fan-out of a few tasks, eight samples of every variant
        dict(name="fan-out, eight samples each", kind="attend", heads=20, kv=20, dim=64, act="f16", cache="bf16", groups=64, items=8, prefix=1193, own=300),
        # requests behind one common preamble, grouped heads
        dict(name="requests behind a preamble", kind="attend", heads=32, kv=8, dim=128, act="bf16", cache="bf16", groups=1, items=64, prefix=8191, own=500),
        # many readers of one long document: the products are what counts
        dict(name="many readers of a document", kind="attend", heads=32, kv=8, dim=128, act="f16", cache="f16", groups=1, items=256, prefix=32768, own=250),
        # groups of very different sizes and lengths, some of one request
        dict(name="ragged groups", kind="attend", heads=16, kv=4, dim=128, act="bf16", cache="bf16", groups=21, items=33, prefix=4999, own=777, ragged=True),
        # five tokens each of sequences under verification: the tokens of a sequence share what it holds
        dict(name="draft tokens", kind="attend", heads=32, kv=8, dim=128, act="f16", cache="f16", groups=24, items=5, prefix=4096, own=5),
        # a reference run in 32 bits
        dict(name="samples in 32 bits", kind="attend", heads=20, kv=5, dim=64, act="f32", cache="f32", groups=3, items=6, prefix=1501, own=97),
        # a short prompt's rows for three more samples, smallest grid model
        dict(name="fork, short prompt", kind="copy", what="fork", planes=8, heads=4, dim=64, cache="bf16", seqs=4, moves=3, rows=190),
        # a long prompt's rows for fifteen more samples, large grid model
        dict(name="fork, sixteen samples", kind="copy", what="fork", planes=24, heads=20, dim=64, cache="bf16", seqs=16, moves=15, rows=1502),
        # beams take each other's places: every place from any other, rows of their own alone
        dict(name="beams reordered", kind="copy", what="reorder", planes=24, heads=5, dim=64, cache="f16", seqs=32, moves=32, rows=233),
        # sequences that are left move into the places of ended ones
        dict(name="sequences compacted", kind="copy", what="compact", planes=16, heads=16, dim=64, cache="bf16", seqs=192, moves=77, rows=700),
    ]


def draw(rng: random.Random) -> dict:
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    if rng.random() < 0.67:
        heads, kv, dim, forms = rng.choice([(4, 4, 64, 0), (12, 12, 64, 0), (20, 20, 64, 0), (20, 5, 64, 1), (16, 4, 128, 1), (32, 8, 128, 1), (32, 32, 128, 1), (16, 1, 128, 1)])
        act, cache = rng.choice([("f16", "bf16"), ("bf16", "bf16")] if forms == 0 else [("f16", "f16"), ("bf16", "bf16"), ("f16", "bf16"), ("f32", "f32")])
        c = dict(kind="attend", heads=heads, kv=kv, dim=dim, act=act, cache=cache, groups=log(1, 64), items=log(1, 256), prefix=log(1, 32768), own=log(1, 931))
        if rng.random() < 0.5:
            c["ragged"] = True
        for key in ("groups", "items", "prefix"):
            while _cost(c) > 1.0 and c[key] > 1:
                c[key] = c[key] * 3 // 4
        return c
    what = rng.choice(["fork", "reorder", "compact"])
    c = dict(kind="copy", what=what, planes=2 * rng.choice([2, 4, 8, 12]), heads=rng.choice([1, 4, 5, 8, 16, 20]), dim=rng.choice([64, 128]),
             cache=rng.choice(["f16", "bf16", "f32"]), rows=log(1, 2048))
    c["seqs"] = log(2, 256)
    c["moves"] = c["seqs"] - 1 if what == "fork" else c["seqs"] if what == "reorder" else rng.randint(1, max(1, c["seqs"] // 2))
    while _cost(c) > 1.0 and c["rows"] > 1:
        c["rows"] = c["rows"] * 3 // 4
    while _cost(c) > 1.0 and c["planes"] > 2:
        c["planes"] -= 2
    return c


# ---------------------------------------------------------------------------
# sizes: functions of the case alone, so that every seed asks for the same amount of work
# ---------------------------------------------------------------------------
def _pitch(rows: int) -> int:
    """Rows of a sequence in the cache: 16 modulo 32, as sessions lay it out."""
    return rows + (16 - rows) % 32


def _group_sizes(c: dict) -> list[int]:
    """Items of every group, the first as many as the case says."""
    if c.get("ragged"):
        return [max(1, c["items"] * (g * 5 % 7 + 1) // 7) if g else c["items"] for g in range(c["groups"])]
    return [c["items"]] * c["groups"]


def _prefix_lengths(c: dict) -> list[int]:
    """Shared rows of every group, the first as many as the case says."""
    return [max(1, c["prefix"] - (g * 389 % (1 + 2 * c["prefix"] // 3))) for g in range(c["groups"])]


def _draft(c: dict) -> bool:
    """The items of a group are the next tokens of one sequence."""
    return c["own"] == c["items"] and c["items"] > 1


def _own_lengths(c: dict) -> list[int]:
    """Rows of its own that every item reads."""
    if _draft(c):
        return [i + 1 for n in _group_sizes(c) for i in range(n)]
    return [c["own"] - (i * 131 % (c["own"] + 1)) for i in range(sum(_group_sizes(c)))]


def _moves(c: dict) -> np.ndarray:
    """[n][4]: sequence read, sequence written, first row, end row."""
    n, rows = c["moves"], c["rows"]
    r = random.Random(3)
    if c["what"] == "fork":
        return np.array([[0, d, 0, rows] for d in range(1, n + 1)], np.int32)
    if c["what"] == "reorder":
        src = [r.randrange(c["seqs"]) for _ in range(n)]
        return np.array([[s, d, 5, 5 + rows] for d, s in enumerate(src) if s != d] or [[0, 1, 5, 5 + rows]], np.int32)
    places = r.sample(range(c["seqs"]), 2 * n)
    return np.array([[max(p), min(p), 0, max(1, rows - r.randrange(1 + rows // 2))] for p in zip(places[:n], places[n:])], np.int32)


def work(case: dict) -> dict:
    c = case
    size = {"f16": 2, "bf16": 2, "f32": 4}
    if c["kind"] == "copy":
        m = _moves(c).astype(np.int64)
        row = c["planes"] * c["heads"] * c["dim"] * size[c["cache"]]
        read = {}
        for s, _, b, e in m.tolist():
            lo, hi = read.get(s, (b, e))
            read[s] = (min(lo, b), max(hi, e))
        return {"bytes": float(row * (int((m[:, 3] - m[:, 2]).sum()) + sum(e - b for b, e in read.values()))), "flops": 0.0}
    sizes, prefix, mine = _group_sizes(c), _prefix_lengths(c), _own_lengths(c)
    n = sum(sizes)
    rows = sum(prefix) + (sum(sizes) if _draft(c) else sum(mine))
    seen = sum(a * b for a, b in zip(sizes, prefix)) + sum(mine)
    return {"bytes": float(2 * n * c["heads"] * c["dim"] * size[c["act"]] + 2 * rows * c["kv"] * c["dim"] * size[c["cache"]]),
            "flops": 4.0 * seen * c["heads"] * c["dim"]}


def _cost(c: dict) -> float:
    """Work and memory of a case against the largest listed ones (1.0: as large)."""
    w = work(c)
    size = 4 if c["cache"] == "f32" else 2
    if c["kind"] == "copy":
        return max(w["bytes"] / 3.0e9, c["planes"] * c["seqs"] * c["heads"] * _pitch(c["rows"] + 5) * c["dim"] * size / 4.5e9)
    n = sum(_group_sizes(c))
    held = 2 * n * c["kv"] * _pitch(c["prefix"] + c["own"]) * c["dim"] * size if not _sparse(c) else 0
    scores = 4 * c["heads"] * n * c["prefix"]
    keys = 8 * c["groups"] * c["kv"] * c["prefix"] * c["dim"] + 8 * n * c["kv"] * c["own"] * c["dim"]
    return max(w["bytes"] / 1.5e9, w["flops"] / (1.4e11 if c["act"] != "f32" else 2e10), held / 6e9, scores / 1.5e9, keys / 4e9)


def _sparse(c: dict) -> bool:
    """Long shared parts are kept in sequences of their own, ahead of the items' short ones (a cache is one pitch wide: the
    items' rows then begin at 0)."""
    return c["groups"] * c["prefix"] + sum(_group_sizes(c)) * c["own"] < sum(_group_sizes(c)) * (c["prefix"] + c["own"]) // 4 and not _draft(c)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def prepare(case: dict, seed: int) -> dict:
    c = case
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = DTYPES[c["cache"]]
    if c["kind"] == "copy":
        shape = (c["planes"], c["seqs"], c["heads"], _pitch(c["rows"] + 5), c["dim"])
        return {"case": c, "cache": torch.randn(shape, device=DEVICE, dtype=dtype, generator=g), "moves": _moves(c)}
    sizes, prefix, mine = _group_sizes(c), _prefix_lengths(c), _own_lengths(c)
    n = sum(sizes)
    first = np.concatenate([[0], np.cumsum(sizes)])
    group_of = np.repeat(np.arange(len(sizes)), sizes)
    if _draft(c):
        # one sequence a group; the items' rows follow the shared ones
        seqs, group_seq, item_seq = len(sizes), np.arange(len(sizes)), group_of
        begin = np.array(prefix)[group_of]
    elif _sparse(c):
        # shared rows cut out of one long sequence each, the items' rows several sequences to a pitch
        per = max(1, (c["prefix"] + c["own"]) // (c["own"] + 1))
        seqs, group_seq = len(sizes) + -(-n // per), np.arange(len(sizes))
        item_seq, begin = len(sizes) + np.arange(n) // per, np.arange(n) % per * c["own"]
    else:
        # every item has a sequence; the shared rows are in the first one's, the others leave that room empty
        seqs, group_seq, item_seq, begin = n, first[:-1], np.arange(n), np.array(prefix)[group_of]
    pitch = _pitch(c["prefix"] + c["own"])

    def ints(a):
        return torch.tensor(np.asarray(a), dtype=torch.int32, device=DEVICE)

    def rows():
        return torch.randn((seqs, c["kv"], pitch, c["dim"]), device=DEVICE, dtype=dtype, generator=g)

    q = torch.randn((n, c["heads"], c["dim"]), device=DEVICE, generator=g) * 2.0     # a few keys stand out, as trained heads have it
    return {"case": c, "q": q.to(DTYPES[c["act"]]), "k": rows(), "v": rows(),
            "group_first": ints(first), "group_seq": ints(group_seq), "group_len": ints(prefix),
            "item_seq": ints(item_seq), "item_begin": ints(begin), "item_end": ints(begin + np.array(mine)),
            "max_group": max(sizes), "max_prefix": max(prefix), "max_own": max(mine)}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state: dict):
    if state["case"]["kind"] == "copy":
        if own:
            from mdlarc_scale_b200 import copy_cache_rows
            copy_cache_rows(state["cache"], state["moves"])
        else:
            _plain_copy(state["cache"], state["moves"])
        cache = state["cache"]
        return cache.view(torch.int32 if cache.dtype == torch.float32 else torch.int16)     # copies are equal to the bit
    if own:
        from mdlarc_scale_b200 import prefix_attention
        s = state
        return prefix_attention(s["q"], s["k"], s["v"], s["group_first"], s["group_seq"], s["group_len"], s["item_seq"], s["item_begin"],
                                s["item_end"], max_group=s["max_group"], max_prefix=s["max_prefix"], max_own=s["max_own"])
    return _plain_attention(state)


def _plain_copy(cache: torch.Tensor, moves: np.ndarray) -> None:
    """All rows are read before the first is written."""
    m = torch.from_numpy(moves).to(cache.device).long()
    n = m[:, 3] - m[:, 2]
    total = int((moves[:, 3] - moves[:, 2]).sum())
    of = torch.repeat_interleave(torch.arange(len(moves), device=cache.device), n, output_size=total)
    row = torch.arange(total, device=cache.device) - (torch.cumsum(n, 0) - n)[of] + m[of, 2]
    cache[:, m[of, 1], :, row] = cache[:, m[of, 0], :, row]


def _plain_attention(s: dict) -> torch.Tensor:
    """Scores of the shared rows group by group (groups padded to the largest), of the own rows item by item, joined by their
    maxima and sums."""
    q, k, v = s["q"].float(), s["k"], s["v"]
    n, heads, dim = q.shape
    kv = k.shape[1]
    rep, dev = heads // kv, q.device
    scale = dim ** -0.5
    qg = q.view(n, kv, rep, dim)
    first, length = s["group_first"].long(), s["group_len"].long()
    item = torch.arange(n, device=dev)
    group = torch.bucketize(item, first[1:], right=True)
    place = item - first[group]
    # shared rows
    padded = torch.zeros((len(length), s["max_group"], kv, rep, dim), device=dev)
    padded[group, place] = qg
    keys = k[s["group_seq"].long(), :, :s["max_prefix"]].float()
    score = torch.einsum("gikrd,gkpd->gkirp", padded, keys) * scale
    hidden = torch.arange(s["max_prefix"], device=dev)[None, :] >= length[:, None]
    score.masked_fill_(hidden[:, None, None, None, :], -math.inf)
    top = score.amax(-1)
    score.sub_(top.clamp_min(-1e30)[..., None]).exp_()
    total = score.sum(-1)
    values = v[s["group_seq"].long(), :, :s["max_prefix"]].float()
    mixed = torch.einsum("gkirp,gkpd->gkird", score, values)
    top, total, mixed = (x.transpose(1, 2)[group, place] for x in (top, total, mixed))       # [n, kv, rep, ...]
    if s["max_own"]:
        # own rows
        begin, end = s["item_begin"].long(), s["item_end"].long()
        row = begin[:, None] + torch.arange(s["max_own"], device=dev)
        hidden = row >= end[:, None]
        row = row.clamp_max(k.shape[2] - 1)[:, None, :]
        seq, head = s["item_seq"].long()[:, None, None], torch.arange(kv, device=dev)[None, :, None]
        score = torch.einsum("nkrd,nkpd->nkrp", qg, k[seq, head, row].float()) * scale
        score.masked_fill_(hidden[:, None, None, :], -math.inf)
        own_top = score.amax(-1)
        score.sub_(own_top.clamp_min(-1e30)[..., None]).exp_()
        both = torch.maximum(top, own_top)
        a, b = (top - both).exp(), (own_top - both).exp()
        total = total * a + score.sum(-1) * b
        mixed = mixed * a[..., None] + torch.einsum("nkrp,nkpd->nkrd", score, v[seq, head, row].float()) * b[..., None]
    return (mixed / total[..., None]).view(n, heads, dim).to(s["q"].dtype)


def exact(case: dict, seed: int):
    """softmax(q K^T / sqrt(dim)) V over an item's shared and own rows together, item by item in 64 bits.  Copies have no
    computed values: the pass returns their bits."""
    if case["kind"] == "copy":
        return None
    s = prepare(case, seed)
    sizes, prefix, mine = _group_sizes(case), _prefix_lengths(case), _own_lengths(case)
    begin, item_seq, group_seq = s["item_begin"].tolist(), s["item_seq"].tolist(), s["group_seq"].tolist()
    rep = case["heads"] // case["kv"]
    out, i = [], 0
    for g, size in enumerate(sizes):
        shared = [x[group_seq[g], :, :prefix[g]].double() for x in (s["k"], s["v"])]
        for _ in range(size):
            keys, values = (torch.cat([p, x[item_seq[i], :, begin[i]:begin[i] + mine[i]].double()], 1) for p, x in zip(shared, (s["k"], s["v"])))
            score = torch.matmul(s["q"][i].double().view(case["kv"], rep, -1), keys.transpose(1, 2)) / math.sqrt(case["dim"])
            out.append(torch.matmul(torch.softmax(score, -1), values).reshape(case["heads"], case["dim"]))
            i += 1
    return torch.stack(out)
