"""The operators that decode several tokens a step, on numpy arrays through the
device C ABI, and their definitions in 64 bits (see tokens.py for the
arithmetic behind the tolerances)."""

import ctypes as C

import numpy as np

import mlvc_hip
from tokens import Padded, f64

ALL = (1 << 64) - 1


# ------------------------------------------------------------ what is seen

def window_seen(nq, nk, causal, window, sinks):
    """[queries, keys]: the last query stands at the last key."""
    place = np.arange(nq)[:, None] + nk - nq
    j = np.arange(nk)[None, :]
    seen = (np.abs(place - j) < window) | (j < sinks) if window else np.ones((nq, nk), bool)
    return seen & (j <= place) if causal else seen


def tree(rng, n, near=8):
    """Ancestor masks of a random tree whose draft 0 follows the context."""
    masks = []
    for i in range(n):
        masks.append((masks[int(rng.integers(max(0, i - near), i))] if i else 0) | 1 << i)
    return masks


def depths(masks, drafts):
    there = (1 << drafts) - 1
    return [bin(m & there & ~(1 << i)).count("1") for i, m in enumerate(masks)]


def drafts_seen(length, masks, window, sinks):
    """[drafts, length]: masks of all of a stream's drafts (at most 64 of them)."""
    n = len(masks)
    past = length - n
    depth = depths(masks, n)
    seen = np.zeros((n, max(length, 0)), bool)
    for i in range(n):
        for j in range(length):
            d = j - past
            place = past + depth[d] if d >= 0 else j
            seen[i, j] = (d < 0 or masks[i] >> d & 1) and (not window or past + depth[i] - place < window or place < sinks)
    return seen


def masked64(q, k, v, scale, seen, tops=None):
    """(result, tolerance) of q [queries, q_heads, dim] on k, v [keys, kv_heads, dim] by what each
    query sees. Weights are off by 2^-11 of themselves or, of FP16 values, by 2^-37 of the largest;
    with `tops`, the rows' largest magnitudes [keys, kv_heads], the weight is taken with the row's
    scale, and by 2^-37 of the largest such product."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    nq, heads, dim = q.shape
    group = heads // max(k.shape[1], 1)
    out, tol = np.zeros_like(q), np.full(q.shape, 2.0 ** -25)
    for h in range(heads):
        for i in range(nq):
            see = np.flatnonzero(seen[i])
            if see.size == 0:
                continue
            kk, vv = k[see, h // group], v[see, h // group]
            with np.errstate(all="ignore"):
                s = kk @ q[i, h] * scale
                # FP32 products and sums of dim terms, then the exponent's own rounding.
                ds = (np.abs(kk) @ np.abs(q[i, h])) * abs(scale) * (dim + 4) * 2.0 ** -24 + np.abs(s) * 2.0 ** -22 + 2.0 ** -21
                p = np.exp(s - s.max())
                w = p / p.sum()
                o = w @ vv
                size = np.abs(vv)
                err = w * (2.0 ** -11 + 2 * ds)
                if tops is None:
                    err = err + 2.0 ** -37 / p.sum()
                else:
                    tol[i, h] += see.size * 2.0 ** -37 * (p * tops[see, h // group]).max() / p.sum()
            out[i, h] = o
            tol[i, h] += np.abs(o) * 2.0 ** -11 + err @ (size + np.abs(o)) + (see.size + 8) * 2.0 ** -24 * (w @ size)
    return out, tol


# ------------------------------------------------------------ plan

class Plan:
    """kv_plan on buffers that stay, and the same by a list of free pages and one stream after the other."""

    def __init__(self, dev, streams, pages, page_size, width, window=0, sinks=0, order=None):
        self.dev, self.streams, self.pages, self.page, self.width = dev, streams, pages, page_size, width
        self.window, self.sinks = window, sinks
        self.table = [[-1] * width for _ in range(streams)]
        self.back = [0] * streams  # entries of a row in use
        self.free = list(range(pages)) if order is None else [int(p) for p in order]
        self.d_table = dev.put(np.full((streams, max(width, 1)), -1, np.int32))
        self.d_held = dev.put(np.zeros((max(streams, 1), 2), np.int32))
        self.d_free, self.d_count = dev.put(np.array(self.free + [0], np.int32)), dev.put(np.array([pages], np.int32))
        self.d_lengths, self.d_starts, self.d_lacking = (dev.put(np.full(n, 77, np.int32)) for n in (streams + 1, streams + 1, 1))

    def desc(self, past, fresh, tokens, seen=None, positions=True):
        """Descriptor of a call on new arrays (or device addresses that stay)."""
        at = lambda a, t: a if a is None or not isinstance(a, (list, np.ndarray)) else self.dev.put(np.asarray(a, t))  # noqa: E731
        self.slots, self.positions = (self.dev.put(np.full(tokens + 4, 77, np.int32)) for _ in range(2))
        return mlvc_hip.KvPlan(
            streams=self.streams, pages=self.pages, page_size=self.page, tokens=tokens, window=self.window, sinks=self.sinks,
            table=self.d_table, table_stride=self.width, held=self.d_held, free_pages=self.d_free, free_count=self.d_count,
            past=at(past, np.int32), fresh=at(fresh, np.int32), seen=at(seen, np.uint64), lengths=self.d_lengths,
            starts=self.d_starts, slots=self.slots, positions=self.positions if positions else None, lacking=self.d_lacking)

    def host(self, past, fresh, tokens, seen=None):
        """The definition; returns what the call writes."""
        page, sink_pages = self.page, -(-self.sinks // self.page) if self.window else 0
        past = [0 if f < 0 else max(p, 0) for p, f in zip(past, fresh)]
        fresh = [max(f, 0) for f in fresh]
        back = []
        for n, row in enumerate(self.table):
            keep = -(-past[n] // page)
            first = max(sink_pages, max(past[n] - self.window + 1, 0) // page) if self.window else 0
            for e in [e for e in range(self.width) if e >= keep] + list(range(sink_pages, min(first, keep, self.width))):
                if row[e] >= 0:
                    back.append(row[e])
                    row[e] = -1
        self.free += back[::-1]
        lengths, starts, slots, positions, lacking, short = [], [0], [], [], 0, False
        for n, row in enumerate(self.table):
            all_tokens = past[n] + fresh[n]
            fits = all_tokens <= self.width * page
            begin = min(-(-past[n] // page), self.back[n])
            need = [e for e in range(begin, -(-all_tokens // page))] if fits else []
            short |= len(need) > len(self.free)
            served = fits and (not need or not short)
            if served:
                for e in need:
                    row[e] = self.free.pop()
            self.back[n] = need[-1] + 1 if served and need else begin
            lacking += not served
            lengths.append(past[n] + (fresh[n] if served else 0))
            starts.append(starts[-1] + fresh[n])
            for i in range(fresh[n]):
                at = past[n] + i
                slots.append(row[at // page] * page + at % page if served else -1)
                positions.append(past[n] + i)
                if seen is not None and len(positions) <= tokens:
                    m = int(seen[len(positions) - 1]) & (1 << min(fresh[n], 64)) - 1 & ~(1 << i)
                    positions[-1] = past[n] + bin(m).count("1")
        cut = lambda a, fill: (a + [fill] * tokens)[:tokens]  # noqa: E731
        return {"table": self.table, "free": self.free, "lengths": lengths, "starts": starts, "slots": cut(slots, -1),
                "positions": cut(positions, 0), "lacking": lacking}

    def compare(self, want, tokens, positions=True):
        get = lambda at, n: self.dev.get(at, (n,), np.int32).tolist()  # noqa: E731
        assert get(self.d_table, self.streams * max(self.width, 1)) == [e for row in want["table"] for e in (row or [-1])]
        count = get(self.d_count, 1)[0]
        assert count == len(want["free"]) and get(self.d_free, self.pages + 1)[:count] == want["free"]
        assert get(self.d_lengths, self.streams + 1) == want["lengths"] + [77]
        assert get(self.d_starts, self.streams + 1) == want["starts"]
        assert get(self.d_lacking, 1) == [want["lacking"]]
        assert get(self.slots, tokens + 4) == want["slots"] + [77] * 4
        assert get(self.positions, tokens + 4) == (want["positions"] if positions else [77] * tokens) + [77] * 4
        pages = [e for row in want["table"] for e in row if e >= 0] + want["free"]
        assert sorted(pages) == sorted(set(pages)) and len(pages) == self.pages  # none lost, none held twice

    def step(self, past, fresh, tokens=None, seen=None, positions=True):
        tokens = sum(max(f, 0) for f in fresh) if tokens is None else tokens
        mlvc_hip.kv_plan(self.desc(past, fresh, tokens, seen, positions))
        want = self.host(past, fresh, tokens, seen)
        self.compare(want, tokens, positions)
        return want


# ------------------------------------------------------------ attention

class Window:
    """Packed sequences under a window."""

    def __init__(self, prompt, window, sinks):
        self.prompt = prompt
        self.desc = mlvc_hip.WindowAttention(prompt=prompt.desc, window=window, sinks=sinks)

    def run(self, stream=None):
        mlvc_hip.attention_window(self.desc, stream)
        return self.prompt.out.get()


class Drafts:
    """Drafts of each stream, rows of q one stream after the other, on a cache."""

    def __init__(self, cache, q, counts, masks, table, lengths, scale, window=0, sinks=0, longest=None, longest_q=None,
                 extra=0, shift=0, starts=None):
        dev = cache.dev
        self.cache, self.out = cache, Padded(dev, np.full(q.shape, np.nan, np.float16), extra, shift)
        self.q = Padded(dev, q, extra, shift)
        table = np.asarray(table, np.int32)
        self.lengths = dev.put(np.asarray(lengths, np.int32))
        self.desc = mlvc_hip.DraftAttention(
            cache=C.pointer(cache.desc), streams=len(counts), q_heads=q.shape[1], q_tokens=q.shape[0],
            longest_q=max(1, max(counts, default=1)) if longest_q is None else longest_q, q=self.q.at, out=self.out.at,
            q_stride=self.q.stride, out_stride=self.out.stride,
            starts=dev.put(np.asarray(np.concatenate([[0], np.cumsum(counts)]) if starts is None else starts, np.int32)),
            seen=None if masks is None else dev.put(np.asarray(masks, np.uint64)), table=dev.put(table),
            table_stride=table.shape[1], lengths=self.lengths, longest=max(lengths, default=0) if longest is None else longest,
            window=window, sinks=sinks, scale=scale)
        need = mlvc_hip.attention_drafts_workspace_bytes(self.desc)
        if need:
            # NaN throughout, so that a partial that is read without having been written shows.
            self.desc.workspace = dev.put(np.full(need, 0xFF, np.uint8))
            self.desc.workspace_bytes = need

    def run(self, stream=None):
        mlvc_hip.attention_drafts(self.desc, stream)
        return self.out.get()


def keep(cache, table, counts, lengths, kept, stream=None):
    """kv_keep; the new lengths. kept: [streams][kept_stride]."""
    dev = cache.dev
    table, kept = np.asarray(table, np.int32), np.asarray(kept, np.int32)
    out = dev.put(np.full(len(counts) + 1, 77, np.int32))
    desc = mlvc_hip.KvKeep(cache=C.pointer(cache.desc), streams=len(counts), table=dev.put(table), table_stride=table.shape[1],
                           starts=dev.put(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)),
                           lengths=dev.put(np.asarray(lengths, np.int32)), kept=dev.put(kept), kept_stride=kept.shape[1],
                           lengths_out=out)
    mlvc_hip.kv_keep(desc, stream)
    got = dev.get(out, (len(counts) + 1,), np.int32).tolist()
    assert got[-1] == 77
    return got[:-1]


class Contexts:
    """Streams with contexts of random rows in a cache whose pages are handed out in any order."""

    def __init__(self, dev, rng, make_cache, kind, heads, dim, page, lengths, spread=1.0):
        used = [max(1, -(-n // page)) for n in lengths]
        order = rng.permutation(sum(used) + 2)
        self.cache = make_cache(dev, kind, sum(used) + 2, page, heads, dim)
        self.table = np.full((len(lengths), max(used)), -1, np.int32)
        self.k, self.v, at = [], [], 0
        for i, (n, pages) in enumerate(zip(lengths, used)):
            self.table[i, :pages] = order[at:at + pages]
            at += pages
            k, v = (rng.standard_normal((n, heads, dim)).astype(np.float16) for _ in range(2))
            v *= np.float16(spread)
            if n:
                self.cache.write(k, v, self.slots(i, np.arange(n)))
            self.k.append(k)
            self.v.append(v)

    def slots(self, i, places):
        places = np.asarray(places)
        return self.table[i, places // self.cache.page_size] * self.cache.page_size + places % self.cache.page_size


def tops_of(v, kind):
    return None if kind == mlvc_hip.KV_F16 else np.abs(f64(v)).max(-1)
