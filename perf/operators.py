"""Performance cases of the token operators: attention over the latents of a
video codec, with the cache that carries them from frame to frame.

A frame's latents are tokens: 12x20, 23x40 or 68x120 of them at 1/16 of
320x192, 640x368 and 1920x1088. Frames that are there already go through
prompt attention in one pass; symbols decoded one by one go through token
attention against a paged cache, whose rows are quantised as they are
written. Queries and keys are normalised per head and rotated by their
position before either.

Each operator is here in its plain form (elementary torch operations in 32
bits, rounded once) and as a call of the device C ABI through mlvc_hip.
"""

from __future__ import annotations

import ctypes as C
import math
import pathlib
import sys

import torch

REPO = pathlib.Path(__file__).resolve().parents[1]

own = False

KINDS = {"f16": 0, "e4m3": 1, "int8": 2}  # cache types
LEVELS = {"e4m3": 448.0, "int8": 127.0}   # largest stored magnitude
EPS = 1e-6


# ------------------------------------------------------------------- cases

def listed():
    return [
        # Norm and rotation of one new token of each of 8 streams: latency.
        _rotate("rotate_8", 8, 16, 4, 64, 64, "half", True),
        # A 1080p frame's latents, half of the head rotated in adjacent pairs.
        _rotate("rotate_8160", 8160, 32, 8, 128, 64, "pairs", True),
        # One new token of each of 64 streams into an INT8 cache, and back.
        _cache("cache_64x1", "int8", 8, 128, 16, 64, 1, 0),
        # A chunk of four 1080p streams into an E4M3 cache, and the whole
        # context read back for prompt attention. Pages of 48 tokens.
        _cache("cache_4x1020", "e4m3", 8, 128, 48, 4, 1020, 1019),
        # One 320x192 frame: 240 tokens, few tiles.
        _prompt("prompt_240", 16, 4, 64, True, "240"),
        # Ragged frames of several streams packed together, one of a single token.
        _prompt("prompt_packed", 16, 4, 128, True, "920,240,1,2040,517,920,1333,64"),
        # A 1080p frame, causal: matrix-bound.
        _prompt("prompt_8160", 16, 4, 128, True, "8160"),
        # A chunk of 920 queries against itself and all that came before,
        # in streams of different age, heads of 64.
        _prompt("prompt_chunk", 16, 16, 64, True, "920,460", "4600,3001"),
        # One stream, one short context: latency.
        _token("token_1x920", "int8", 16, 4, 64, 16, 1, 920, 920),
        # One stream with eight 1080p frames behind it: one long axis to split.
        _token("token_1x65280", "e4m3", 32, 8, 128, 64, 1, 65280, 65280),
        # 64 streams of every age up to a 1080p frame.
        _token("token_64x8160", "int8", 32, 8, 128, 16, 64, 1, 8160),
        # 16 streams, unquantised cache, as many key heads as query heads.
        _token("token_16x3001_f16", "f16", 16, 16, 64, 32, 16, 920, 3001),
    ]


def _rotate(name, tokens, q_heads, kv_heads, dim, rot, layout, norm, scaling=1.0):
    c = {"kind": "rotate", "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "rot": rot,
         "layout": layout, "norm": norm, "scaling": scaling}
    return dict(c, name=name) if name else c


def _cache(name, kind, heads, dim, page, streams, new, past):
    c = {"kind": "cache", "type": kind, "heads": heads, "dim": dim, "page": page, "streams": streams, "new": new,
         "past": past}
    return dict(c, name=name) if name else c


def _prompt(name, q_heads, kv_heads, dim, causal, queries, keys=""):
    c = {"kind": "prompt", "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "causal": causal, "queries": queries,
         "keys": keys or queries}
    return dict(c, name=name) if name else c


def _token(name, kind, q_heads, kv_heads, dim, page, streams, shortest, longest):
    c = {"kind": "token", "type": kind, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "page": page,
         "streams": streams, "shortest": shortest, "longest": longest}
    return dict(c, name=name) if name else c


HEADS = ((16, 4), (32, 8), (16, 16), (8, 1), (12, 4), (16, 1), (10, 2), (8, 8))


def draw(rng):
    """One more call of the same ranges: 1 to 8160 tokens a pass, contexts to 65280, every head layout and cache type."""
    def spread(lo, hi):
        return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))

    while True:
        kind = rng.choice(("rotate", "cache", "prompt", "token"))
        q_heads, kv_heads = rng.choice(HEADS)
        dim = rng.choice((64, 128))
        if kind == "rotate":
            dim = rng.choice((64, 96, 128))
            c = _rotate(None, spread(1, 8160), q_heads, kv_heads, dim, rng.choice((dim, dim // 2, dim // 4)),
                        rng.choice(("half", "pairs")), rng.random() < 0.75, rng.choice((1.0, 1.0, 4.0)))
        elif kind == "cache":
            streams = spread(1, 64)
            c = _cache(None, rng.choice(("int8", "e4m3", "f16")), kv_heads, rng.choice((64, 96, 128)),
                       rng.choice((16, 32, 48, 64)), streams, spread(1, 4080 // streams + 1), rng.choice((0, spread(1, 2000))))
        elif kind == "prompt":
            n = rng.choice((1, 1, 2, 3, 5, 8))
            queries = [spread(1, 8160 // n) for _ in range(n)]
            keys = queries if rng.random() < 0.6 else [q + spread(1, 2000) for q in queries]
            c = _prompt(None, q_heads, kv_heads, dim, rng.random() < 0.8, ",".join(map(str, queries)),
                        ",".join(map(str, keys)))
        else:
            longest = spread(16, 65280)
            c = _token(None, rng.choice(("int8", "e4m3", "f16")), q_heads, kv_heads, dim, rng.choice((16, 32, 48, 64)),
                       spread(1, 64), rng.choice((1, longest, max(1, longest // 3))), longest)
        w = work(c)
        plain = 4.0 * _scores(c)
        if w["bytes"] <= 5.5e8 and w["flops"] <= 2.7e11 and plain <= 5e9:
            return c


def _ints(text):
    return [int(v) for v in text.split(",")]


def _scores(c):
    """Scores that the plain form materialises."""
    if c["kind"] == "prompt":
        return c["q_heads"] * sum(_ints(c["queries"])) * sum(_ints(c["keys"]))
    return c["q_heads"] * c["streams"] * c["longest"] if c["kind"] == "token" else 0


def _ages(c):
    """Context lengths of the streams, evenly from the shortest to the longest."""
    n = c["streams"]
    if n == 1:
        return [c["longest"]]
    return [c["shortest"] + (c["longest"] - c["shortest"]) * i // (n - 1) for i in range(n)]


def _row_bytes(kind, dim):
    """Bytes of one cached row of one head: its values and its scale."""
    return 2 * dim if kind == "f16" else dim + 4


def work(c):
    if c["kind"] == "rotate":
        rows = c["tokens"] * (c["q_heads"] + c["kv_heads"])
        return {"bytes": rows * c["dim"] * 4 + c["tokens"] * 4 + c["rot"] * 4, "flops": rows * (c["dim"] * 4 + c["rot"] * 3)}
    if c["kind"] == "cache":
        wrote, read = c["streams"] * c["new"], c["streams"] * (c["new"] + c["past"])
        rows = (wrote + read) * c["heads"] * 2
        return {"bytes": rows * (2 * c["dim"] + _row_bytes(c["type"], c["dim"])) + 4 * (wrote + read),
                "flops": rows * c["dim"] * 2}
    if c["kind"] == "prompt":
        queries, keys = _ints(c["queries"]), _ints(c["keys"])
        pairs = sum(q * k - (q * (q - 1) // 2 if c["causal"] else 0) for q, k in zip(queries, keys))
        rows = 2 * sum(queries) * c["q_heads"] + 2 * sum(keys) * c["kv_heads"]
        return {"bytes": rows * c["dim"] * 2, "flops": 4 * c["dim"] * c["q_heads"] * pairs}
    tokens, n = sum(_ages(c)), c["streams"]
    return {"bytes": 2 * tokens * c["kv_heads"] * _row_bytes(c["type"], c["dim"]) + 4 * n * c["q_heads"] * c["dim"]
            + 4 * n + 4 * sum(-(-t // c["page"]) for t in _ages(c)),
            "flops": 4 * c["dim"] * c["q_heads"] * tokens}


# ------------------------------------------------------------------ inputs

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFFFFFF)


def _normal(g, shape, std=1.0):
    return torch.empty(shape, device="cuda").normal_(0, std, generator=g).half()


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return _i32(at)


def _frequencies(c):
    """Radians a position of each pair, base 10000, positions interpolated by the scaling, in FP64."""
    i = torch.arange(c["rot"] // 2, dtype=torch.float64, device="cuda")
    return 10000.0 ** (-2.0 * i / c["rot"]) / c["scaling"]


def _heavy_rows(g, shape):
    """Keys and values as a cache meets them: rows of different magnitude."""
    x = torch.empty(shape, device="cuda").normal_(0, 1, generator=g)
    x *= torch.empty((*shape[:-1], 1), device="cuda").uniform_(0.25, 2.0, generator=g)
    return x.half()


def _inputs(c, seed):
    g = _generator(seed)
    if c["kind"] == "rotate":
        return {"q": _normal(g, (c["tokens"], c["q_heads"], c["dim"]), 1.5),
                "k": _normal(g, (c["tokens"], c["kv_heads"], c["dim"]), 1.5),
                "wq": _normal(g, (c["dim"],), 0.1) + 1, "wk": _normal(g, (c["dim"],), 0.1) + 1,
                "positions": torch.randint(0, 65280, (c["tokens"],), generator=g, device="cuda", dtype=torch.int32),
                "freqs": _frequencies(c)}
    if c["kind"] == "prompt":
        tq, tk = sum(_ints(c["queries"])), sum(_ints(c["keys"]))
        return {"q": _normal(g, (tq, c["q_heads"], c["dim"])), "k": _normal(g, (tk, c["kv_heads"], c["dim"])),
                "v": _normal(g, (tk, c["kv_heads"], c["dim"]))}
    if c["kind"] == "cache":
        ages, heads = [c["new"] + c["past"]] * c["streams"], c["heads"]
        s = {"k": _heavy_rows(g, (c["streams"] * c["new"], heads, c["dim"])),
             "v": _heavy_rows(g, (c["streams"] * c["new"], heads, c["dim"]))}
    else:
        order = torch.randperm(c["streams"], generator=g, device="cuda").tolist()
        ages, heads = [_ages(c)[i] for i in order], c["kv_heads"]
        s = {"q": _normal(g, (c["streams"], c["q_heads"], c["dim"])), "lengths": _i32(ages)}
    # A pool of pages handed out in any order; what a table has past a
    # stream's last page is the pool's first page.
    used = [-(-n // c["page"]) for n in ages]
    width, total = max(max(used), 1), sum(used) + 1
    pages = torch.randperm(total, generator=g, device="cuda", dtype=torch.int32)
    ends = torch.tensor(used, device="cuda").cumsum(0)
    column = torch.arange(width, device="cuda")
    at = (ends - torch.tensor(used, device="cuda"))[:, None] + column
    s["table"] = torch.where(column < torch.tensor(used, device="cuda")[:, None], pages[at.clamp(max=total - 1)], 0).int().contiguous()
    s["past_k"] = _heavy_rows(g, (total, heads, c["page"], c["dim"]))
    s["past_v"] = _heavy_rows(g, (total, heads, c["page"], c["dim"]))
    s["ages"] = ages
    if c["kind"] == "cache":
        position = torch.arange(c["new"] + c["past"], device="cuda")
        slots = s["table"][:, position // c["page"]] * c["page"] + position % c["page"]
        s["read_slots"] = slots.reshape(-1).int().contiguous()
        s["write_slots"] = slots[:, c["past"]:].reshape(-1).int().contiguous()
    return s


# ------------------------------------------------------------- plain forms

def _quantise(x, kind):
    """Rows of FP16 -> (stored values as uint8 or FP16, FP32 scale of each row)."""
    if kind == "f16":
        return x, None
    x = x.float()
    largest = x.abs().amax(-1, keepdim=True)
    level = torch.full_like(largest, LEVELS[kind])
    scale = largest / level
    # x * level is exact, so the quotient's ties are, and round to even.
    q = x * level / torch.where(largest > 0, largest, 1.0)
    q = torch.round(q).to(torch.int8) if kind == "int8" else q.to(torch.float8_e4m3fn)
    return q.view(torch.uint8), scale[..., 0]


def _values(q, kind):
    return q.float() if kind == "f16" else q.view(torch.int8 if kind == "int8" else torch.float8_e4m3fn).float()


def _rotated(x, w, s):
    x = x.float()
    if s["norm"]:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
    # The phase of a far position does not fit 24 bits: it is reduced to one
    # turn in 64 bits before the 32-bit part.
    turns = s["positions"].double()[:, None] * (s["freqs"] / (2 * math.pi))
    angle = ((turns - torch.floor(turns)) * (2 * math.pi)).float()[:, None, :]
    cos, sin = torch.cos(angle), torch.sin(angle)
    part, rest = x[..., :s["rot"]], x[..., s["rot"]:]
    if s["layout"] == "half":
        a, b = part.chunk(2, -1)
        part = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = part[..., 0::2], part[..., 1::2]
        part = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([part, rest], -1).half()


def _plain_rotate(s):
    return {"q": _rotated(s["q"], s["wq"], s), "k": _rotated(s["k"], s["wk"], s)}


def _kept(s, name):
    """New rows quantised into the cache, and all rows asked for read back."""
    kind, page = s["type"], s["page"]
    wrote, read = s["write_slots"].long(), s["read_slots"].long()
    rows, scale = _quantise(s[name], kind)
    cache, scales = s["cache_" + name], s["scale_" + name]
    cache[wrote // page, :, wrote % page] = rows
    back = _values(cache[read // page, :, read % page], kind)
    if scales is not None:
        scales[wrote // page, :, wrote % page] = scale
        back = back * scales[read // page, :, read % page][..., None]
    return back.half()


def _plain_cache(s):
    return {"k": _kept(s, "k"), "v": _kept(s, "v")}


def _weights(scores, seen):
    """Softmax over the last axis of what is seen; rows that see nothing weigh nothing."""
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, 1.0, total)


def _plain_prompt(s):
    group = s["q_heads"] // s["kv_heads"]
    q, k, v = s["q"].float().transpose(0, 1), s["k"].float().transpose(0, 1), s["v"].float().transpose(0, 1)
    of_q = torch.repeat_interleave(torch.arange(s["n"], device="cuda"), s["q_lengths"], output_size=q.shape[1])
    of_k = torch.repeat_interleave(torch.arange(s["n"], device="cuda"), s["k_lengths"], output_size=k.shape[1])
    seen = of_q[:, None] == of_k[None, :]
    if s["causal"]:
        # Places counted from the end of each sequence: the last query sees the last key.
        to_end_q = s["q_starts"][1:][of_q] - torch.arange(q.shape[1], device="cuda")
        to_end_k = s["k_starts"][1:][of_k] - torch.arange(k.shape[1], device="cuda")
        seen &= to_end_k[None, :] >= to_end_q[:, None]
    q = q.reshape(s["kv_heads"], group * q.shape[1], s["dim"])
    p = torch.matmul(q, k.transpose(1, 2).contiguous()) * s["scale"]
    p = _weights(p.view(s["kv_heads"], group, *seen.shape), seen)
    o = torch.matmul(p.view(s["kv_heads"], -1, seen.shape[1]), v.contiguous())
    return o.view(s["q_heads"], -1, s["dim"]).transpose(0, 1).half().contiguous()


def _context(s, name):
    """[streams, heads, tokens, dim] of the pages in the table, unpacked."""
    pages = s["table"].long()
    x = _values(s["cache_" + name][pages], s["type"])
    if s["scale_" + name] is not None:
        x = x * s["scale_" + name][pages][..., None]
    return x.transpose(1, 2).reshape(x.shape[0], s["kv_heads"], -1, s["dim"])


def _plain_token(s):
    n, heads, dim = s["q"].shape[0], s["kv_heads"], s["dim"]
    q = s["q"].float().view(n, heads, -1, dim)
    p = torch.matmul(q, _context(s, "k").transpose(2, 3).contiguous()) * s["scale"]
    seen = torch.arange(p.shape[-1], device="cuda") < s["lengths"][:, None, None, None]
    return torch.matmul(_weights(p, seen), _context(s, "v")).view(n, -1, dim).half()


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
    if kind == "rotate":
        s["out"] = {"q": torch.empty_like(s["q"]), "k": torch.empty_like(s["k"])}
        nq, nk = s["q"][0].numel(), s["k"][0].numel()
        d = hip.QkNormRope(tokens=s["q"].shape[0], q_heads=s["q"].shape[1], k_heads=s["k"].shape[1], head_dim=s["dim"],
                           q=_at(s["q"]), k=_at(s["k"]), q_out=_at(s["out"]["q"]), k_out=_at(s["out"]["k"]),
                           q_stride=nq, k_stride=nk, q_out_stride=nq, k_out_stride=nk,
                           q_weight=_at(s["wq"]) if s["norm"] else None, k_weight=_at(s["wk"]) if s["norm"] else None,
                           eps=EPS, positions=_at(s["positions"]), freqs=_at(s["freqs"]), rot_dim=s["rot"],
                           interleaved=int(s["layout"] == "pairs"), rot_scale=1.0)
        s["call"] = lambda stream: hip.qk_norm_rope(d, stream)
    elif kind == "cache":
        shape = (s["read_slots"].numel(), s["heads"], s["dim"])
        s["out"] = {n: torch.empty(shape, dtype=torch.float16, device="cuda") for n in ("k", "v")}
        row = s["heads"] * s["dim"]
        cache = _kv_cache(hip, s)
        wrote = hip.KvRows(k=_at(s["k"]), v=_at(s["v"]), k_stride=row, v_stride=row, slots=_at(s["write_slots"]),
                           tokens=s["write_slots"].numel())
        read = hip.KvRows(k=_at(s["out"]["k"]), v=_at(s["out"]["v"]), k_stride=row, v_stride=row,
                          slots=_at(s["read_slots"]), tokens=s["read_slots"].numel())
        s["call"] = lambda stream: (hip.kv_write(cache, wrote, stream), hip.kv_read(cache, read, stream))
    elif kind == "prompt":
        s["out"] = torch.empty_like(s["q"])
        nq, nk = s["q"][0].numel(), s["k"][0].numel()
        d = hip.PromptAttention(sequences=s["n"], q_heads=s["q_heads"], kv_heads=s["kv_heads"], head_dim=s["dim"],
                                q=_at(s["q"]), k=_at(s["k"]), v=_at(s["v"]), out=_at(s["out"]),
                                q_stride=nq, k_stride=nk, v_stride=nk, out_stride=nq,
                                q_starts=_at(s["q_starts"]), k_starts=_at(s["k_starts"]), q_tokens=s["q"].shape[0],
                                k_tokens=s["k"].shape[0], longest_q=s["longest_q"], causal=int(s["causal"]),
                                scale=s["scale"])
        s["call"] = lambda stream: hip.attention_prompt(d, stream)
    else:
        s["out"] = torch.empty_like(s["q"])
        nq = s["q"][0].numel()
        cache = _kv_cache(hip, s)
        d = hip.TokenAttention(cache=C.pointer(cache), streams=s["q"].shape[0], q_heads=s["q"].shape[1],
                               q=_at(s["q"]), out=_at(s["out"]), q_stride=nq, out_stride=nq, table=_at(s["table"]),
                               table_stride=s["table"].shape[1], lengths=_at(s["lengths"]), longest=s["longest"],
                               scale=s["scale"])
        need = hip.attention_token_workspace_bytes(d)
        s["workspace"] = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
        d.workspace, d.workspace_bytes = _at(s["workspace"]), need
        s["call"] = lambda stream: hip.attention_token(d, stream)


# ------------------------------------------------------------ prepare, run

def prepare(case, seed):
    s = dict(case)
    s.update(_inputs(case, seed))
    kind = case["kind"]
    if kind in ("prompt", "token"):
        s["scale"] = 1.0 / math.sqrt(case["dim"])
    if kind == "prompt":
        queries, keys = _ints(case["queries"]), _ints(case["keys"])
        s.update(n=len(queries), q_starts=_starts(queries), k_starts=_starts(keys), longest_q=max(queries),
                 q_lengths=_i32(queries), k_lengths=_i32(keys))
    elif kind in ("cache", "token"):
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
    """Each operator from its definition in 64 bits, one sequence or stream at a time."""
    return globals()["_exact_" + case["kind"]](case, _inputs(case, seed))


def _exact_rotate(c, s):
    def rotated(x, w):
        x = x.double()
        if c["norm"]:
            x = w.double() * x / torch.sqrt((x * x).sum(-1, keepdim=True) / c["dim"] + EPS)
        z = torch.polar(torch.ones(c["tokens"], c["rot"] // 2, dtype=torch.float64, device="cuda"),
                        s["positions"].double().outer(s["freqs"]))[:, None]
        half = c["rot"] // 2
        first = torch.arange(half, device="cuda") * (1 if c["layout"] == "half" else 2)
        second = first + (half if c["layout"] == "half" else 1)
        turned = torch.complex(x[..., first], x[..., second]) * z
        y = x.clone()
        y[..., first], y[..., second] = turned.real, turned.imag
        return y

    return {"q": rotated(s["q"], s["wq"]), "k": rotated(s["k"], s["wk"])}


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
    exponent = torch.floor(torch.log2(units.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(exponent - 3)
    return torch.round(units / step) * step * scale


def _exact_cache(c, s):
    out = {}
    for name in ("k", "v"):
        new = _stored64(s[name], c["type"]).view(c["streams"], c["new"], c["heads"], c["dim"])
        past = _stored64(s["past_" + name], c["type"])
        streams = []
        for i in range(c["streams"]):
            rows = past[s["table"][i].long()].transpose(1, 2).reshape(-1, c["heads"], c["dim"])[:c["past"]]
            streams += [rows, new[i]]
        out[name] = torch.cat(streams)
    return out


def _attend64(q, k, v, scale, causal):
    """[queries, q heads, dim] on [keys, kv heads, dim]."""
    out = torch.zeros_like(q)
    group = q.shape[1] // k.shape[1]
    last = torch.arange(q.shape[0], device="cuda") + (k.shape[0] - q.shape[0])
    for h in range(q.shape[1]):
        s = q[:, h] @ k[:, h // group].t() * scale
        if causal:
            s.masked_fill_(torch.arange(k.shape[0], device="cuda")[None, :] > last[:, None], -math.inf)
        out[:, h] = torch.nan_to_num(torch.softmax(s, -1), nan=0.0) @ v[:, h // group]
    return out


def _exact_prompt(c, s):
    out, q0, k0 = [], 0, 0
    for nq, nk in zip(_ints(c["queries"]), _ints(c["keys"])):
        out.append(_attend64(s["q"][q0:q0 + nq].double(), s["k"][k0:k0 + nk].double(), s["v"][k0:k0 + nk].double(),
                             1 / math.sqrt(c["dim"]), c["causal"]))
        q0, k0 = q0 + nq, k0 + nk
    return torch.cat(out)


def _exact_token(c, s):
    out = []
    for i, n in enumerate(s["ages"]):
        k, v = (_stored64(s["past_" + name][s["table"][i].long()], c["type"]).transpose(1, 2).reshape(
            -1, c["kv_heads"], c["dim"])[:n] for name in ("k", "v"))
        out.append(_attend64(s["q"][i:i + 1].double(), k, v, 1 / math.sqrt(c["dim"]), False))
    return torch.cat(out)
