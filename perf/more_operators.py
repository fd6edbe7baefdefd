"""Performance cases of the operators that decode several tokens a step in
bounded memory: page tables and slots planned on the GPU, attention with a
sliding window and sinks (the first tokens stay visible), attention of trees
of drafted tokens on the paged cache, and the move of the drafts that are kept.

A stream's latents are tokens, 240 to 8160 of them a frame. Symbols are drafted
several at a time, as a tree: every draft attends to its stream's context and
to the drafts it follows, and once the entropy decoder has told which path was
right, the rows of that path move behind the context. Old frames leave by the
window, and their pages go back to the pool.

Each operator is here in its plain form (elementary torch operations in 32
bits, rounded once) and as a call of the device C ABI through mlvc_hip.
"""

from __future__ import annotations

import ctypes as C
import math
import pathlib
import sys

import numpy as np
import torch

REPO = pathlib.Path(__file__).resolve().parents[1]

own = False

KINDS = {"f16": 0, "e4m3": 1, "int8": 2}  # cache types
LEVELS = {"e4m3": 448.0, "int8": 127.0}   # largest stored magnitude


# ------------------------------------------------------------------- cases

def listed():
    return [
        # One new token of each of 64 streams of every age: latency.
        _plan("plan_64x1", 64, 16, 1, 8160, 1, False, 0, 0),
        # Ragged prompts of 64 streams, some of them ended, behind a window of
        # one 640x368 frame whose pages go back.
        _plan("plan_64x2040", 64, 16, 0, 4080, 2040, False, 920, 4),
        # Trees of 8 drafts, four kept: latency.
        _keep("keep_8x8", "int8", 8, 128, 16, 8, 240, 8, 4),
        # Trees of 64 drafts of 64 streams, unquantised, half of their drafts kept.
        _keep("keep_64x64", "f16", 8, 128, 48, 64, 240, 64, 31),
        # One 320x192 frame, each token sees four rows of 20 and the first tokens.
        _window("window_240", 16, 4, 64, True, 80, 4, "240"),
        # Ragged frames packed together, each token sees those around it.
        _window("window_packed", 16, 16, 64, False, 240, 0, "920,2040,1,517,920,1333"),
        # Four 1080p frames of one stream, a window of 1024 tokens and 4 sinks.
        _window("window_32640", 16, 4, 128, True, 1024, 4, "32640"),
        # One token of one stream under a window: latency.
        _drafts("drafts_1x1", "int8", 16, 4, 64, 16, 1, 8160, 8160, 1, 920, 4),
        # One token of each of 64 streams, windows of half a 1080p frame.
        _drafts("drafts_64x1", "e4m3", 32, 8, 128, 64, 64, 2040, 8160, 1, 4080, 4),
        # A tree of 16 on one stream with eight 1080p frames behind it.
        _drafts("drafts_1x16", "e4m3", 32, 8, 128, 64, 1, 65280, 65280, 16, 0, 0),
        # Trees of 16 on 64 streams of every age up to a 1080p frame.
        _drafts("drafts_64x16", "int8", 32, 8, 128, 16, 64, 16, 8160, 16, 0, 0),
        # Trees of 64, unquantised cache, as many key heads as query heads.
        _drafts("drafts_16x64_f16", "f16", 16, 16, 64, 32, 16, 920, 3001, 64, 2040, 16),
    ]


def _named(name, c):
    return dict(c, name=name) if name else c


def _plan(name, streams, page, shortest, longest, fresh, tree, window, sinks):
    return _named(name, {"kind": "plan", "streams": streams, "page": page, "shortest": shortest, "longest": longest,
                         "fresh": fresh, "tree": tree, "window": window, "sinks": sinks})


def _keep(name, kind, heads, dim, page, streams, past, drafts, kept):
    return _named(name, {"kind": "keep", "type": kind, "heads": heads, "dim": dim, "page": page, "streams": streams,
                         "past": past, "drafts": drafts, "kept": kept})


def _window(name, q_heads, kv_heads, dim, causal, window, sinks, queries, keys=""):
    return _named(name, {"kind": "window", "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "causal": causal,
                         "window": window, "sinks": sinks, "queries": queries, "keys": keys or queries})


def _drafts(name, kind, q_heads, kv_heads, dim, page, streams, shortest, longest, drafts, window, sinks):
    """Contexts of shortest to longest tokens, the drafts among them."""
    return _named(name, {"kind": "drafts", "type": kind, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
                         "page": page, "streams": streams, "shortest": shortest, "longest": longest,
                         "drafts": drafts, "window": window, "sinks": sinks})


HEADS = ((16, 4), (32, 8), (16, 16), (8, 1), (12, 4), (16, 1), (10, 2), (8, 8))
PAGES = (16, 32, 48, 64)


def draw(rng):
    """One more call of the same ranges: 1 to 64 drafts, contexts to 65280, prompts to 32640, every head layout and cache type."""
    def spread(lo, hi):
        return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))

    while True:
        kind = rng.choice(("plan", "keep", "window", "drafts"))
        q_heads, kv_heads = rng.choice(HEADS)
        dim = rng.choice((64, 128))
        window, sinks = rng.choice((0, spread(1, 4080), spread(16, 2040))), rng.choice((0, spread(1, 64)))
        if kind == "plan":
            streams, tree = spread(1, 256), rng.random() < 0.4
            c = _plan(None, streams, rng.choice(PAGES), rng.choice((0, 1, 240)), spread(240, 8160),
                      spread(1, 64) if tree else spread(1, min(8160, 130560 // streams)), tree, window, sinks)
        elif kind == "keep":
            drafts = spread(2, 64)
            c = _keep(None, rng.choice(("int8", "f16")), kv_heads, rng.choice((64, 96, 128)), rng.choice(PAGES),
                      spread(1, 64), spread(1, 240), drafts, rng.randint(1, (drafts + 1) // 2))
        elif kind == "window":
            n = rng.choice((1, 1, 2, 3, 5, 8))
            queries = [spread(1, 32640 // n) for _ in range(n)]
            keys = queries if rng.random() < 0.6 else [q + spread(1, 2000) for q in queries]
            c = _window(None, q_heads, kv_heads, dim, rng.random() < 0.7, window or spread(1, 4080), sinks,
                        ",".join(map(str, queries)), ",".join(map(str, keys)))
        else:
            drafts = rng.choice((1, spread(2, 64)))
            longest = spread(max(drafts, 16), 65280)
            c = _drafts(None, rng.choice(("int8", "e4m3", "f16")), q_heads, kv_heads, dim, rng.choice(PAGES),
                        spread(1, 64), rng.choice((drafts, longest, max(drafts, longest // 3))), longest, drafts, window, sinks)
        w = work(c)
        if w["bytes"] <= 5.5e8 and w["flops"] <= 2.7e11 and _gathered(c) <= 5.4e8:
            return c


def _ints(text):
    return [int(v) for v in text.split(",")]


def _gathered(c):
    """Values that the plain form unpacks of the contexts, and scores that it makes."""
    if c["kind"] != "drafts":
        return 0
    return c["streams"] * c["longest"] * max(c["kv_heads"] * c["dim"], c["q_heads"] * c["drafts"])


def _ages(c):
    """Context lengths of the streams, evenly from the shortest to the longest."""
    n = c["streams"]
    if n == 1:
        return [c["longest"]]
    return [c["shortest"] + (c["longest"] - c["shortest"]) * i // (n - 1) for i in range(n)]


def _fresh(c):
    """New tokens of the streams, evenly up to the most; of 16 streams one has none, and one has ended."""
    n, most = c["streams"], c["fresh"]
    if most == 1:
        return [1] * n
    return [-1 if i % 16 == 15 else 0 if i % 16 == 7 else 1 + (most - 1) * (i + 1) // n for i in range(n)]


def _row_bytes(kind, dim):
    """Bytes of one cached row of one head: its values and its scale."""
    return 2 * dim if kind == "f16" else dim + 4


def _union(lo, hi, first):
    """Keys in [lo, hi) or [0, first)."""
    width = np.maximum(hi - lo, 0)
    return width + first - np.where(width > 0, np.clip(np.minimum(first, hi) - lo, 0, None), 0)


def _window_pairs(c, nq, nk):
    place = np.arange(nq, dtype=np.int64) + nk - nq
    end = np.clip(place + 1, 0, nk) if c["causal"] else np.full(nq, nk, dtype=np.int64)
    lo, hi = np.maximum(place - c["window"] + 1, 0), np.clip(np.minimum(end, place + c["window"]), 0, None)
    return int(_union(lo, hi, np.minimum(c["sinks"], end)).sum())


def work(c):
    if c["kind"] == "plan":
        # A stream's lengths and what it holds, in and out; a slot and a position a token; the pages handed out.
        tokens = sum(max(f, 0) for f in _fresh(c))
        return {"bytes": 36 * c["streams"] + tokens * (16 if c["tree"] else 8) + 8 * (tokens // c["page"]), "flops": 4 * tokens}
    if c["kind"] == "keep":
        rows = c["streams"] * (c["kept"] - 1) * c["heads"] * 2
        return {"bytes": 2 * rows * _row_bytes(c["type"], c["dim"]) + c["streams"] * (4 * c["kept"] + 16), "flops": rows}
    if c["kind"] == "window":
        queries, keys = _ints(c["queries"]), _ints(c["keys"])
        pairs = sum(_window_pairs(c, q, k) for q, k in zip(queries, keys))
        rows = 2 * sum(queries) * c["q_heads"] + 2 * sum(keys) * c["kv_heads"]
        return {"bytes": rows * c["dim"] * 2, "flops": 4 * c["dim"] * c["q_heads"] * pairs}
    n, drafts = c["streams"], c["drafts"]
    past = np.array(_ages(c), dtype=np.int64) - drafts
    lo = np.maximum(past - c["window"] + 1, 0) if c["window"] else np.zeros_like(past)
    rows = int(_union(lo, past, np.minimum(c["sinks"], past)).sum())
    # A tree of n drafts is about log n deep: its part of the pairs is small and counted as that.
    pairs = drafts * rows + n * drafts * (1 + int(math.log2(drafts)))
    return {"bytes": 2 * (rows + n * drafts) * c["kv_heads"] * _row_bytes(c["type"], c["dim"])
            + 4 * n * drafts * c["q_heads"] * c["dim"] + 8 * n * drafts + 4 * n + 4 * rows // c["page"],
            "flops": 4 * c["dim"] * c["q_heads"] * pairs}


# ------------------------------------------------------------------ inputs

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFFFFFF)


def _normal(g, shape, std=1.0):
    return torch.empty(shape, device="cuda").normal_(0, std, generator=g).half()


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(lengths):
    return _i32(np.concatenate([[0], np.cumsum(lengths)]).tolist())


def _heavy_rows(g, shape):
    """Keys and values as a cache meets them: rows of different magnitude."""
    x = torch.empty(shape, device="cuda").normal_(0, 1, generator=g)
    x *= torch.empty((*shape[:-1], 1), device="cuda").uniform_(0.25, 2.0, generator=g)
    return x.half()


def _trees(seed, counts):
    """Ancestor masks of random trees, one after the other: draft 0 follows the
    context, every other one a draft among the eight before it."""
    rng = np.random.default_rng(seed & 0x7FFFFFFFFFFF)
    masks = []
    for n in counts:
        tree = []
        for i in range(n):
            up = tree[int(rng.integers(max(0, i - 8), i))] if i else 0
            tree.append(up | 1 << i)
        masks += tree
    return torch.from_numpy(np.array(masks, dtype=np.uint64).view(np.int64)).cuda()


def _pool(g, used, width):
    """Tables of streams that hold `used` pages each, of a pool handed out in any order (-1 past a
    stream's last), and the pool's pages that are free."""
    total = sum(used)
    spare = len(used) * width - total
    pages = torch.randperm(total + spare, generator=g, device="cuda", dtype=torch.int32)
    count = torch.tensor(used, device="cuda")
    column = torch.arange(width, device="cuda")
    at = (count.cumsum(0) - count)[:, None] + column
    held = column < count[:, None]
    return torch.where(held, pages[at.clamp(max=total + spare - 1)], -1).int().contiguous(), pages[total:]


def _inputs(c, seed):
    g = _generator(seed)
    if c["kind"] == "window":
        tq, tk = sum(_ints(c["queries"])), sum(_ints(c["keys"]))
        return {"q": _normal(g, (tq, c["q_heads"], c["dim"])), "k": _normal(g, (tk, c["kv_heads"], c["dim"])),
                "v": _normal(g, (tk, c["kv_heads"], c["dim"]))}
    page = c["page"]
    if c["kind"] == "plan":
        n = c["streams"]
        order = torch.randperm(n, generator=g, device="cuda").tolist()
        past = [_ages(c)[i] for i in order]
        order = torch.randperm(n, generator=g, device="cuda").tolist()
        fresh = [_fresh(c)[i] for i in order]
        used = [-(-p // page) for p in past]
        width = -(-(c["longest"] + c["fresh"]) // page)
        table, free = _pool(g, used, width)
        s = {"past": _i32(past), "fresh": _i32(fresh), "table": table, "width": width, "pages": n * width,
             "held": torch.stack([torch.zeros(n, dtype=torch.int32, device="cuda"), _i32(used)], 1).contiguous(),
             "free_count": _i32([free.numel()])}
        # A stack of all pages; what lies above its top means nothing.
        s["free_pages"] = torch.full((s["pages"],), -1, dtype=torch.int32, device="cuda")
        s["free_pages"][:free.numel()] = free
        new = [max(f, 0) for f in fresh]
        s["tokens"] = -(-max(sum(new), 1) // 8) * 8  # rows of a batch, the last few of them padding
        if c["tree"]:
            s["seen"] = torch.zeros(s["tokens"], dtype=torch.int64, device="cuda")
            s["seen"][:sum(new)] = _trees(seed, new)
        return s
    if c["kind"] == "keep":
        ages, heads, drafts = [c["past"] + c["drafts"]] * c["streams"], c["heads"], c["drafts"]
        # Paths down the trees: the root, then drafts further on than the path is long.
        rng = np.random.default_rng(seed & 0x7FFFFFFFFFFF)
        kept = [[0] + sorted(rng.choice(np.arange(c["kept"], drafts), c["kept"] - 1, replace=False).tolist())
                for _ in range(c["streams"])]
        s = {"kept": _i32(kept)}
    else:
        order = torch.randperm(c["streams"], generator=g, device="cuda").tolist()
        ages, heads, drafts = [_ages(c)[i] for i in order], c["kv_heads"], c["drafts"]
        s = {"q": _normal(g, (c["streams"] * drafts, c["q_heads"], c["dim"])), "seen": _trees(seed, [drafts] * c["streams"])}
    used = [-(-n // page) for n in ages]
    s["table"], _ = _pool(g, used, max(used))
    s["lengths"], s["starts"], s["ages"] = _i32(ages), _starts([drafts] * c["streams"]), ages
    total = c["streams"] * max(used)
    s["past_k"] = _heavy_rows(g, (total, heads, page, c["dim"]))
    s["past_v"] = _heavy_rows(g, (total, heads, page, c["dim"]))
    return s


# ------------------------------------------------------------- plain forms

def _quantise(x, kind):
    """Rows of FP16 -> (stored values as uint8 or FP16, FP32 scale of each row)."""
    if kind == "f16":
        return x, None
    x = x.float()
    largest = x.abs().amax(-1, keepdim=True)
    scale = largest / torch.full_like(largest, LEVELS[kind])
    # x * level is exact, so the quotient's ties are, and round to even.
    q = x * LEVELS[kind] / torch.where(largest > 0, largest, 1.0)
    q = torch.round(q).to(torch.int8) if kind == "int8" else q.to(torch.float8_e4m3fn)
    return q.view(torch.uint8), scale[..., 0]


def _values(q, kind):
    return q.float() if kind == "f16" else q.view(torch.int8 if kind == "int8" else torch.float8_e4m3fn).float()


def _weights(scores, seen):
    """Softmax over the last axis of what is seen; rows that see nothing weigh nothing."""
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, 1.0, total)


def _bits(masks):
    """[drafts, 64]: whether a draft sees the j-th of its stream."""
    return (masks[:, None] >> torch.arange(64, device="cuda")) & 1


def _depths(masks, index):
    """How many other drafts a draft, the index-th of its stream, sees."""
    bits = _bits(masks)
    return bits.sum(1) - bits.gather(1, index[:, None])[:, 0]


def _entries(first, last):
    """(row, entry) of the ranges [first, last) of each row, one after the other; ranges [rows] or [rows, k]."""
    first, last = (t.reshape(t.shape[0], -1) for t in (first, last))
    count = (last - first).clamp(min=0).reshape(-1)
    of = torch.repeat_interleave(torch.arange(count.numel(), device="cuda"), count)
    inside = torch.arange(of.numel(), device="cuda") - (count.cumsum(0) - count)[of]
    return of // first.shape[1], first.reshape(-1)[of] + inside


def _plain_plan(s):
    page, table, free = s["page"], s["table"], s["free_pages"]
    fresh, (front, back) = s["fresh"].long(), s["held"].long().unbind(1)
    past = torch.where(fresh < 0, 0, s["past"].long())
    lengths = past + fresh.clamp(min=0)
    kept, need = (past + page - 1) // page, (lengths + page - 1) // page
    sinks = torch.full_like(past, -(-s["sinks"] // page) if s["window"] else 0)
    begin = torch.maximum((past - s["window"] + 1).clamp(min=0) // page, sinks) if s["window"] else sinks
    # Pages that go back: sinks not kept, what is behind the context, what is before the window.
    outside = torch.maximum(front, sinks)
    stream, entry = _entries(torch.stack([kept, torch.maximum(kept, outside), outside], 1),
                             torch.stack([torch.minimum(sinks, back), back, torch.minimum(torch.minimum(begin, kept), back)], 1))
    top = s["free_count"].long() + stream.numel()
    free[top - 1 - torch.arange(stream.numel(), device="cuda")] = table[stream, entry]
    table[stream, entry] = -1
    stream, entry = _entries(torch.minimum(back, kept), need)
    table[stream, entry] = free[top - 1 - torch.arange(stream.numel(), device="cuda")]
    s["free_count"].copy_(top - stream.numel())
    s["held"].copy_(torch.stack([torch.maximum(begin, torch.minimum(front, kept)) if s["window"] else front * 0, need], 1))
    starts = torch.cat([past.new_zeros(1), fresh.clamp(min=0).cumsum(0)])
    stream, place = _entries(past, lengths)
    slots = torch.full((s["tokens"],), -1, dtype=torch.int32, device="cuda")
    positions = torch.zeros_like(slots)
    slots[:stream.numel()] = table[stream, place // page] * page + (place % page).int()
    if s["tree"]:
        place = past[stream] + _depths(s["seen"][:stream.numel()], place - past[stream])
    positions[:stream.numel()] = place.int()
    return {"table": table, "held": s["held"], "free_pages": free, "free_count": s["free_count"], "lengths": lengths.int(),
            "starts": starts.int(), "slots": slots, "positions": positions, "lacking": torch.zeros(1, dtype=torch.int32, device="cuda")}


def _kept_out(s, lengths):
    """The cache as it stands after a move: stored values as they are."""
    view = (lambda t: t) if s["type"] == "f16" else (lambda t: t.view(torch.int8))
    out = {"k": view(s["cache_k"]), "v": view(s["cache_v"]), "lengths": lengths}
    return out if s["scale_k"] is None else dict(out, k_scale=s["scale_k"], v_scale=s["scale_v"])


def _plain_keep(s):
    page, table = s["page"], s["table"].long()
    past = (s["lengths"] - (s["starts"][1:] - s["starts"][:-1])).long()[:, None]
    stream = torch.arange(table.shape[0], device="cuda")[:, None]
    source = past + s["kept"].long()
    target = past + torch.arange(s["kept"].shape[1], device="cuda")
    for t in (s["cache_k"], s["cache_v"], s["scale_k"], s["scale_v"]):
        if t is not None:
            t[table[stream, target // page], :, target % page] = t[table[stream, source // page], :, source % page]
    return _kept_out(s, (past[:, 0] + s["kept"].shape[1]).int())


def _plain_window(s):
    queries, keys, window, sinks, dim, heads = _ints(s["queries"]), _ints(s["keys"]), s["window"], s["sinks"], s["dim"], s["kv_heads"]
    out = torch.empty_like(s["q"])
    step, q0, k0 = 1024, 0, 0
    for nq, nk in zip(queries, keys):
        for first in range(0, nq, step):
            # The queries of a block, and the keys that any of them sees.
            count = min(step, nq - first)
            place = torch.arange(first, first + count, device="cuda") + (nk - nq)
            begin = max(0, first + nk - nq - window + 1)
            end = max(min(nk, first + count + nk - nq + (0 if s["causal"] else window - 1)), 0)
            some = min(sinks, nk)
            key = torch.cat([torch.arange(min(some, begin), device="cuda"), torch.arange(begin, max(end, begin, min(some, nk)), device="cuda")])
            key = key[key < nk]
            seen = ((place[:, None] - key).abs() < window) | (key < sinks)
            if s["causal"]:
                seen &= key <= place[:, None]
            if key.numel() == 0:
                out[q0 + first:q0 + first + count] = 0
                continue
            q = s["q"][q0 + first:q0 + first + count].float().transpose(0, 1).reshape(heads, -1, dim)
            k, v = (s[name][k0 + key].float().transpose(0, 1) for name in ("k", "v"))
            p = torch.matmul(q, k.transpose(1, 2).contiguous()) * s["scale"]
            p = _weights(p.view(heads, -1, *seen.shape), seen).view(heads, -1, key.numel())
            out[q0 + first:q0 + first + count] = torch.matmul(p, v.contiguous()).view(-1, count, dim).transpose(0, 1).half()
        q0, k0 = q0 + nq, k0 + nk
    return out


def _context(s, name):
    """[streams, heads, tokens, dim] of the pages in the table, unpacked."""
    pages = s["table"].long().clamp(min=0)
    x = _values(s["cache_" + name][pages], s["type"])
    if s["scale_" + name] is not None:
        x = x * s["scale_" + name][pages][..., None]
    return x.transpose(1, 2).reshape(x.shape[0], s["kv_heads"], -1, s["dim"])


def _plain_drafts(s):
    n, drafts, heads, dim, window, sinks = s["streams"], s["drafts"], s["kv_heads"], s["dim"], s["window"], s["sinks"]
    k, v = _context(s, "k"), _context(s, "v")
    index = torch.arange(drafts, device="cuda")
    past = (s["lengths"] - drafts).long()
    depth = _depths(s["seen"], index.repeat(n)).view(n, drafts)
    # Places of the keys: a draft's is its depth behind the context.
    j = torch.arange(k.shape[2], device="cuda")
    of = (j - past[:, None]).clamp(0, drafts - 1)
    in_context = j < past[:, None]
    place = torch.where(in_context, j, past[:, None] + depth.gather(1, of))
    seen = in_context[:, None] | (_bits(s["seen"]).view(n, drafts, 64).gather(2, of[:, None].expand(-1, drafts, -1)) > 0)
    seen &= (j < s["lengths"][:, None])[:, None]
    if window:
        seen &= ((past[:, None] + depth)[:, :, None] - place[:, None] < window) | (place < sinks)[:, None]
    q = s["q"].float().view(n, drafts, heads, -1, dim).permute(0, 2, 3, 1, 4).reshape(n, heads, -1, dim)
    p = torch.matmul(q, k.transpose(2, 3).contiguous()) * s["scale"]
    p = _weights(p.view(n, heads, -1, drafts, p.shape[-1]), seen[:, None, None]).view(p.shape)
    o = torch.matmul(p, v).view(n, heads, -1, drafts, dim)
    return o.permute(0, 3, 1, 2, 4).reshape(n * drafts, -1, dim).half()


# ----------------------------------------------------- the framework's calls

def _hip():
    if str(REPO / "mlvc.cpp_amd" / "python") not in sys.path:
        sys.path.insert(0, str(REPO / "mlvc.cpp_amd" / "python"))
    import mlvc_hip

    return mlvc_hip


def _at(t):
    return None if t is None else t.data_ptr()


def _kv_cache(hip, s):
    pages, heads, page, dim = s["cache_k"].shape
    return hip.KvCache(kind=KINDS[s["type"]], pages=pages, page_size=page, heads=heads, head_dim=dim,
                       k=_at(s["cache_k"]), v=_at(s["cache_v"]), k_scale=_at(s["scale_k"]), v_scale=_at(s["scale_v"]))


def _describe(s):
    """The descriptors of a state's buffers, filled once as a program that keeps its buffers fills them."""
    hip = _hip()
    kind = s["kind"]
    if kind == "plan":
        n = s["streams"]
        out = {name: torch.empty(size, dtype=torch.int32, device="cuda") for name, size in (
            ("lengths", n), ("starts", n + 1), ("slots", s["tokens"]), ("positions", s["tokens"]), ("lacking", 1))}
        s["out"] = {name: s[name] for name in ("table", "held", "free_pages", "free_count")} | out
        d = hip.KvPlan(streams=n, pages=s["pages"], page_size=s["page"], tokens=s["tokens"], window=s["window"],
                       sinks=s["sinks"], table=_at(s["table"]), table_stride=s["width"], held=_at(s["held"]),
                       free_pages=_at(s["free_pages"]), free_count=_at(s["free_count"]), past=_at(s["past"]),
                       fresh=_at(s["fresh"]), seen=_at(s.get("seen")), **{name: _at(t) for name, t in out.items()})
        s["call"] = lambda stream: hip.kv_plan(d, stream)
    elif kind == "keep":
        cache = _kv_cache(hip, s)
        lengths = torch.empty_like(s["lengths"])
        s["out"] = _kept_out(s, lengths)
        d = hip.KvKeep(cache=C.pointer(cache), streams=s["streams"], table=_at(s["table"]), table_stride=s["table"].shape[1],
                       starts=_at(s["starts"]), lengths=_at(s["lengths"]), kept=_at(s["kept"]),
                       kept_stride=s["kept"].shape[1], lengths_out=_at(lengths))
        s["call"] = lambda stream: hip.kv_keep(d, stream)
    elif kind == "window":
        queries, keys = _ints(s["queries"]), _ints(s["keys"])
        s["out"] = torch.empty_like(s["q"])
        nq, nk = s["q"][0].numel(), s["k"][0].numel()
        d = hip.WindowAttention(
            prompt=hip.PromptAttention(
                sequences=len(queries), q_heads=s["q_heads"], kv_heads=s["kv_heads"], head_dim=s["dim"], q=_at(s["q"]),
                k=_at(s["k"]), v=_at(s["v"]), out=_at(s["out"]), q_stride=nq, k_stride=nk, v_stride=nk, out_stride=nq,
                q_starts=_at(s["q_starts"]), k_starts=_at(s["k_starts"]), q_tokens=s["q"].shape[0],
                k_tokens=s["k"].shape[0], longest_q=max(queries), causal=int(s["causal"]), scale=s["scale"]),
            window=s["window"], sinks=s["sinks"])
        s["call"] = lambda stream: hip.attention_window(d, stream)
    else:
        s["out"] = torch.empty_like(s["q"])
        row = s["q"][0].numel()
        cache = _kv_cache(hip, s)
        d = hip.DraftAttention(cache=C.pointer(cache), streams=s["streams"], q_heads=s["q_heads"], q_tokens=s["q"].shape[0],
                               longest_q=s["drafts"], q=_at(s["q"]), out=_at(s["out"]), q_stride=row, out_stride=row,
                               starts=_at(s["starts"]), seen=_at(s["seen"]), table=_at(s["table"]),
                               table_stride=s["table"].shape[1], lengths=_at(s["lengths"]), longest=s["longest"],
                               window=s["window"], sinks=s["sinks"], scale=s["scale"])
        need = hip.attention_drafts_workspace_bytes(d)
        s["workspace"] = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
        d.workspace, d.workspace_bytes = _at(s["workspace"]), need
        s["call"] = lambda stream: hip.attention_drafts(d, stream)


# ------------------------------------------------------------ prepare, run

def prepare(case, seed):
    s = dict(case)
    s.update(_inputs(case, seed))
    kind = case["kind"]
    if kind in ("window", "drafts"):
        s["scale"] = 1.0 / math.sqrt(case["dim"])
    if kind == "window":
        s.update(q_starts=_starts(_ints(case["queries"])), k_starts=_starts(_ints(case["keys"])))
    elif kind != "plan":
        for name in ("k", "v"):
            s["cache_" + name], s["scale_" + name] = _quantise(s.pop("past_" + name), case["type"])
    return s


def run(state):
    if not own:
        return globals()["_plain_" + state["kind"]](state)
    if "call" not in state:
        _describe(state)
    state["call"](torch.cuda.current_stream().cuda_stream)
    return state["out"]


# ------------------------------------------------------------------- exact

def exact(case, seed):
    """Each operator from its definition in 64 bits, one sequence, stream or page at a time."""
    return globals()["_exact_" + case["kind"]](case, _inputs(case, seed))


def _exact_plan(c, s):
    page, window = c["page"], c["window"]
    past, fresh, table = s["past"].tolist(), s["fresh"].tolist(), s["table"].tolist()
    stack = s["free_pages"].tolist()
    top = int(s["free_count"])
    back = []
    pages = -(-c["sinks"] // page) if window else 0
    before = []
    for n, row in enumerate(table):
        if fresh[n] < 0:
            past[n] = 0
        keep = -(-past[n] // page)
        first = max(pages, max(past[n] - window + 1, 0) // page) if window else 0
        before.append(first)
        for e in [e for e in range(len(row)) if e >= keep] + [e for e in range(pages, min(first, keep))]:
            if row[e] >= 0:
                back.append(row[e])
                row[e] = -1
    for p in reversed(back):
        stack[top] = p
        top += 1
    lengths, starts, slots, positions, held = [], [0], [], [], []
    for n, row in enumerate(table):
        new = max(fresh[n], 0)
        for i in range(new):
            at = past[n] + i
            if row[at // page] < 0:
                top -= 1
                row[at // page] = stack[top]
            slots.append(row[at // page] * page + at % page)
            others = bin(int(s["seen"][len(positions)]) & 0xFFFFFFFFFFFFFFFF & ~(1 << i)).count("1") if c["tree"] else i
            positions.append(past[n] + others)
        lengths.append(past[n] + new)
        starts.append(starts[-1] + new)
        held.append([before[n], -(-lengths[n] // page)])
    pad = s["tokens"] - len(slots)
    out = {"table": table, "held": held, "free_pages": stack, "free_count": [top], "lengths": lengths, "starts": starts,
           "slots": slots + [-1] * pad, "positions": positions + [0] * pad, "lacking": [0]}
    return {name: _i32(v) for name, v in out.items()}


def _exact_keep(c, s):
    out = {"lengths": _i32([c["past"] + c["kept"]] * c["streams"])}
    table, kept, page = s["table"].tolist(), s["kept"].tolist(), c["page"]
    for name in ("k", "v"):
        rows, scale = _quantise(s["past_" + name], c["type"])
        tensors = [(name, rows.view(torch.int8) if scale is not None else rows.double())]
        tensors += [] if scale is None else [(name + "_scale", scale.double())]
        for key, t in tensors:
            new = t.clone()
            for n, row in enumerate(table):
                for i, draft in enumerate(kept[n]):
                    a, b = c["past"] + draft, c["past"] + i
                    new[row[b // page], :, b % page] = t[row[a // page], :, a % page]
            out[key] = new
    return out


def _attend64(q, k, v, scale, seen):
    """[queries, q heads, dim] on [keys, kv heads, dim], by what each query sees."""
    out = torch.zeros_like(q)
    group = q.shape[1] // k.shape[1]
    for h in range(q.shape[1]):
        p = q[:, h] @ k[:, h // group].t() * scale
        p.masked_fill_(~seen, -math.inf)
        out[:, h] = torch.nan_to_num(torch.softmax(p, -1), nan=0.0) @ v[:, h // group]
    return out


def _exact_window(c, s):
    out, q0, k0 = [], 0, 0
    for nq, nk in zip(_ints(c["queries"]), _ints(c["keys"])):
        k, v = (s[name][k0:k0 + nk].double() for name in ("k", "v"))
        for i in range(0, nq, 2048):
            place = torch.arange(i, min(i + 2048, nq), device="cuda") + (nk - nq)
            # No query of the block sees the keys between the sinks and `first`.
            first = max(0, min(int(place[0]) - c["window"] + 1, nk) - c["sinks"])
            last = min(nk, max(int(place[-1]) + c["window"], c["sinks"], 0))
            key = torch.cat([torch.arange(min(first, c["sinks"]), device="cuda"),
                             torch.arange(min(first, last), last, device="cuda")]).unique()
            away = place[:, None] - key
            seen = (away.abs() < c["window"]) | (key < c["sinks"])[None, :]
            if c["causal"]:
                seen &= away >= 0
            out.append(_attend64(s["q"][q0 + i:q0 + i + len(place)].double(), k[key], v[key], 1 / math.sqrt(c["dim"]), seen))
        q0, k0 = q0 + nq, k0 + nk
    return torch.cat(out)


def _stored64(x, kind):
    """What a row of the cache stands for: the scale is the FP32 value that the cache holds."""
    x = x.double()
    if kind == "f16":
        return x
    top = x.abs().max(-1, keepdim=True).values
    scale = (top / LEVELS[kind]).float().double()
    units = torch.nan_to_num(x * LEVELS[kind] / top, nan=0.0)
    if kind == "int8":
        return torch.round(units) * scale
    # E4M3: four significant bits, steps of 2^-9 below 2^-6, nearest even.
    step = torch.exp2(torch.floor(torch.log2(units.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(units / step) * step * scale


def _exact_drafts(c, s):
    out, m = [], c["drafts"]
    masks = [v & 0xFFFFFFFFFFFFFFFF for v in s["seen"].tolist()]
    for i, n in enumerate(s["ages"]):
        past = n - m
        tree = masks[i * m:(i + 1) * m]
        depth = [bin(t & ~(1 << d)).count("1") for d, t in enumerate(tree)]
        place = torch.tensor(list(range(past)) + [past + d for d in depth], device="cuda")
        seen = torch.ones(m, n, dtype=torch.bool, device="cuda")
        for d, t in enumerate(tree):
            seen[d, past:] = torch.tensor([bool(t >> e & 1) for e in range(m)], device="cuda")
            if c["window"]:
                seen[d] &= (past + depth[d] - place < c["window"]) | (place < c["sinks"])
        k, v = (_stored64(s["past_" + name][s["table"][i].long().clamp(min=0)], c["type"]).transpose(1, 2).reshape(
            -1, c["kv_heads"], c["dim"])[:n] for name in ("k", "v"))
        out.append(_attend64(s["q"][i * m:(i + 1) * m].double(), k, v, 1 / math.sqrt(c["dim"]), seen))
    return torch.cat(out)
