"""Drafts where a context, a list or a number ends: cuts, drafts that do not
count, pages that ran out, the last lengths and the largest scores."""

import ctypes as C

import numpy as np
import pytest

import mlvc_hip
from devmem import Dev
from drafts import ALL, Contexts, Drafts, Plan, Window, depths, drafts_seen, masked64, tops_of, tree, window_seen
from mlvc_hip import KV_E4M3, KV_F16, KV_INT8
from tokens import Cache, Padded, Prompt, f64, stored64, within

pytestmark = pytest.mark.gpu

KINDS = [KV_F16, KV_E4M3, KV_INT8]


@pytest.fixture
def dev():
    d = Dev()
    yield d
    d.close()


def normal(rng, *shape):
    return rng.standard_normal(shape).astype(np.float16)


def check(got, q, k, v, kind, scale, seen, what):
    want, tol = masked64(f64(q), stored64(k, kind), stored64(v, kind), scale, seen, tops_of(v, kind))
    within(got, want, tol, what)


# ------------------------------------------------------------ cuts

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("q_heads,heads,dim,counts,lengths,cuts,window", [
    # Whole contexts: 16 rows, 32, 64, 128; padded heads; value by value.
    (4, 2, 64, [1, 5, 3], [900, 400, 150], [49, 81, 127, 145], 0),
    (4, 2, 128, [8, 5, 3], [900, 400, 150], [60, 118], 500),
    (16, 2, 64, [4, 3, 2] * 44, [300, 130, 97] * 44, [60], 0),
    (4, 1, 128, [16, 5, 6] * 50, [205, 130, 97] * 50, [63], 0),
    (16, 8, 64, [20, 17, 1] * 22, [250, 164, 97] * 22, [50], 0),
    (16, 8, 64, [64, 40, 33, 50, 1] * 8, [170, 150, 164, 196, 133] * 8, [55], 0),
    (4, 2, 96, [7, 5, 3], [900, 400, 150], [60, 17], 0),
    (2, 1, 256, [7, 5, 3], [300, 400, 150], [63], 90),
    (2, 1, 264, [7, 5, 3], [300, 400, 150], [60], 0),
    # Cut over workgroups.
    (4, 2, 64, [3, 1, 9], [2900, 1500, 2175], [2100, 2174, 2075], 0),
    (4, 2, 128, [15, 9, 20], [2700, 1500, 2400], [2130], 0),
    (6, 2, 64, [20, 16, 30], [2700, 1500, 2400], [2162], 0),
    (4, 2, 64, [64, 3, 33], [9000, 3040, 8700], [8300, 8600], 0),
    (4, 2, 96, [9, 1, 30], [2900, 1500, 2175], [2100], 0),
    (2, 1, 264, [2, 1, 3], [2900, 1500, 2175], [2100], 0),
])
def test_tokens_past_longest_are_not_seen(dev, rng, kind, q_heads, heads, dim, counts, lengths, cuts, window):
    """Contexts that `longest` cuts inside the second tile of a step, long before the drafts, with NaN behind the cut."""
    for cut in cuts:
        ctx = Contexts(dev, rng, Cache, kind, heads, dim, 16, lengths)
        bad = np.full((1, heads, dim), np.nan, np.float16)
        for i, n in enumerate(lengths):
            if i % 2 == 0 and n > cut:
                ctx.cache.write(bad, bad, ctx.slots(i, [cut]))
        q = normal(rng, sum(counts), q_heads, dim)
        trees = [tree(rng, n) for n in counts]
        got = Drafts(ctx.cache, q, counts, [m for t in trees for m in t], ctx.table, lengths, dim ** -0.5, window, 4, longest=cut).run()
        at = 0
        for i, (count, n) in enumerate(zip(counts, lengths)):
            if i < 5:
                seen = drafts_seen(n, trees[i], window, 4)[:, :cut]
                check(got[at:at + count], q[at:at + count], ctx.k[i][:cut], ctx.v[i][:cut], kind, dim ** -0.5, seen, f"stream {i} cut at {cut}")
            at += count


# ------------------------------------------------------------ pages that ran out

@pytest.mark.parametrize("streams", [1, 64, 70, 1100])
def test_plan_tells_what_is_placed(dev, rng, streams):
    """Of a short pool and of short rows, also where the streams take several turns."""
    plan = Plan(dev, streams, 2 * streams, 16, 3, order=rng.permutation(2 * streams))
    placed = dev.put(np.full(streams + 1, 77, np.int32))
    length = np.zeros(streams, int)
    short = 0
    for _ in range(5):
        fresh = rng.integers(-1, 30, streams)
        total = int(fresh.clip(0).sum())
        desc = plan.desc(length.tolist(), fresh.tolist(), total)
        desc.placed = placed
        mlvc_hip.kv_plan(desc)
        want = plan.host(length.tolist(), fresh.tolist(), total)
        plan.compare(want, total)
        got = dev.get(placed, (streams + 1,), np.int32)
        past = np.where(fresh < 0, 0, length)
        assert got[-1] == 77 and np.array_equal(got[:-1], np.array(want["lengths"]) - past)
        short += want["lacking"]
        length = np.array(want["lengths"])
    assert short or streams == 1


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 96, 264])
def test_first_drafts_alone_are_placed(dev, rng, kind, dim):
    """`placed` below the drafts of starts: those behind are not computed; above: no more than there are."""
    counts, placed, lengths = [7, 70, 3, 5, 4], [3, 66, 0, 9, -2], [40, 100, 41, 5, 1300]
    ctx = Contexts(dev, rng, Cache, kind, 1, dim, 16, lengths)
    here = [min(max(p, 0), n) for p, n in zip(placed, counts)]
    trees = [tree(rng, min(n, 64)) + [0] * max(n - 64, 0) for n in counts]
    q = normal(rng, sum(counts), 2, dim)
    d = Drafts(ctx.cache, q, counts, [m for t in trees for m in t], ctx.table, lengths, 0.1, longest_q=64)
    d.desc.placed = dev.put(np.array(placed, np.int32))
    got, at = d.run(), 0
    for i, (count, n) in enumerate(zip(counts, lengths)):
        done = min(here[i], 64)
        seen = np.zeros((done, n), bool)
        for r in range(done):
            for j in range(n):
                e = j - (n - here[i])
                seen[r, j] = e < 0 or (e < 64 and trees[i][r] >> e & 1)
        check(got[at:at + done], q[at:at + done], ctx.k[i], ctx.v[i], kind, 0.1, seen, f"stream {i}")
        assert np.isnan(got[at + done:at + count]).all()
        at += count
    new = dev.put(np.full(6, 77, np.int32))
    kept = np.array([[2, 3], [65, 66], [0, 1], [1, 4], [0, 1]], np.int32)
    mlvc_hip.kv_keep(mlvc_hip.KvKeep(cache=C.pointer(ctx.cache.desc), streams=5, table=d.desc.table, table_stride=d.desc.table_stride,
                                     starts=d.desc.starts, lengths=d.lengths, kept=dev.put(kept), kept_stride=2, lengths_out=new,
                                     placed=d.desc.placed))
    assert dev.get(new, (6,), np.int32).tolist() == [38, 35, 41, 2, 1300, 77]
    moved = [{37: 39}, {34: 99}, {}, {0: 1, 1: 4}, {}]
    for i, n in enumerate(lengths):
        order = np.array([moved[i].get(j, j) for j in range(n)])
        for g, x in zip(ctx.cache.read(ctx.slots(i, np.arange(n))), (ctx.k[i], ctx.v[i])):
            want = stored64(x, kind)[order]
            within(g, want, np.abs(want) * (2.0 ** -11 + 2.0 ** -23) + 2.0 ** -25)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("pages,width,window,sinks", [
    (7, 40, 0, 0),      # a pool for fewer tokens than the streams take
    (9, 40, 40, 5),     # the same behind a window
    (40, 3, 0, 0),      # rows of 48 tokens, pages enough
])
def test_loop_that_runs_out_of_pages(dev, rng, kind, pages, width, window, sinks):
    """Plan, write, attend to and keep drafts, captured once and replayed: a stream that gets no pages keeps its
    rows, its length and its rows of out, and goes on once pages are there again."""
    streams, heads, q_heads, dim, page, most = 4, 2, 4, 64, 16, 8
    plan = Plan(dev, streams, pages, page, width, window, sinks, rng.permutation(pages))
    cache = Cache(dev, kind, pages, page, heads, dim)
    put = lambda shape, t: dev.put(np.zeros(shape, t))  # noqa: E731
    tokens = streams * most
    past, fresh, kept, seen, placed = put(streams, np.int32), put(streams, np.int32), put((streams, most), np.int32), put(tokens, np.uint64), put(streams, np.int32)
    x = np.zeros((tokens, heads, dim), np.float16)
    q, k, v = Padded(dev, np.zeros((tokens, q_heads, dim), np.float16)), Padded(dev, x), Padded(dev, x)
    out = Padded(dev, np.full((tokens, q_heads, dim), np.nan, np.float16))
    pd = plan.desc(past, fresh, tokens, seen)
    pd.placed = placed
    rows = mlvc_hip.KvRows(tokens=tokens, k=k.at, v=v.at, k_stride=k.stride, v_stride=v.stride, slots=plan.slots)
    ad = mlvc_hip.DraftAttention(cache=C.pointer(cache.desc), streams=streams, q_heads=q_heads, q_tokens=tokens, longest_q=most,
                                 q=q.at, out=out.at, q_stride=q.stride, out_stride=out.stride, starts=plan.d_starts, seen=seen,
                                 table=plan.d_table, table_stride=width, lengths=plan.d_lengths, longest=width * page,
                                 window=window, sinks=sinks, scale=0.125, placed=placed)
    ad.workspace_bytes = mlvc_hip.attention_drafts_workspace_bytes(ad)
    if ad.workspace_bytes:
        ad.workspace = dev.put(np.full(ad.workspace_bytes, 0xFF, np.uint8))
    kd = mlvc_hip.KvKeep(cache=C.pointer(cache.desc), streams=streams, table=plan.d_table, table_stride=width, starts=plan.d_starts,
                         lengths=plan.d_lengths, kept=kept, kept_stride=most, lengths_out=past, placed=placed)
    stream, graph = C.c_void_p(), C.c_void_p()
    dev.check(dev.lib.mlvc_hip_stream_synchronize(None))
    dev.check(dev.lib.mlvc_hip_stream_create(C.byref(stream)))
    dev.check(dev.lib.mlvc_hip_capture_begin(stream))
    mlvc_hip.kv_plan(pd, stream)
    mlvc_hip.kv_write(cache.desc, rows, stream)
    mlvc_hip.attention_drafts(ad, stream)
    mlvc_hip.kv_keep(kd, stream)
    dev.check(dev.lib.mlvc_hip_capture_end(stream, C.byref(graph)))

    def set_(at, a):
        a = np.ascontiguousarray(a)
        dev.check(dev.lib.mlvc_hip_memcpy_h2d(at, a.ctypes.data, a.nbytes, stream))
        dev.check(dev.lib.mlvc_hip_stream_synchronize(stream))

    length, refused, again, waits = [0] * streams, 0, 0, set()
    held_k, held_v = [np.zeros((0, heads, dim), np.float16) for _ in range(streams)], [np.zeros((0, heads, dim), np.float16) for _ in range(streams)]
    for step in range(40):
        counts = [int(rng.integers(1, most + 1)) for _ in range(streams)]
        if step % 9 == 8:                       # one ends, its pages go to those that wait
            i = int(np.argmax(length))
            counts[i], length[i] = -1, 0
            held_k[i] = held_v[i] = held_k[i][:0]
            waits.discard(i)
        trees = [tree(rng, max(n, 0), 3) for n in counts]
        n_new = sum(max(n, 0) for n in counts)
        qn, kn, vn = normal(rng, tokens, q_heads, dim), normal(rng, tokens, heads, dim), normal(rng, tokens, heads, dim)
        paths = np.full((streams, most), -1, np.int32)
        for i, t in enumerate(trees):
            if t:
                leaf = int(rng.integers(0, len(t)))
                path = [j for j in range(len(t)) if t[leaf] >> j & 1]
                paths[i, :len(path)] = path
        masks = np.array([m for t in trees for m in t] + [0] * (tokens - n_new), np.uint64)
        set_(fresh, np.array(counts, np.int32))
        set_(kept, paths)
        set_(seen, masks)
        for p, a in ((q, qn), (k, kn), (v, vn)):
            set_(p.base, np.concatenate([a.reshape(-1).view(np.uint16), np.full(8, 0x7E00, np.uint16)]))
        set_(out.base, np.full(out.n, 0x7E00, np.uint16))
        dev.check(dev.lib.mlvc_hip_graph_launch(graph, stream))
        dev.check(dev.lib.mlvc_hip_stream_synchronize(stream))
        want = plan.host(length, counts, tokens, masks)
        plan.compare(want, tokens)
        got, at = out.get(), 0
        for i, t in enumerate(trees):
            n = len(t)
            if n and want["lengths"][i] == length[i]:
                assert np.isnan(got[at:at + n]).all()
                refused += 1
                waits.add(i)
            elif n:
                again += i in waits
                waits.discard(i)
                kk, vv = np.concatenate([held_k[i], kn[at:at + n]]), np.concatenate([held_v[i], vn[at:at + n]])
                check(got[at:at + n], qn[at:at + n], kk, vv, kind, 0.125, drafts_seen(length[i] + n, t, window, sinks), f"step {step}, stream {i}")
                path = [d for d in paths[i] if d >= 0]
                held_k[i], held_v[i] = np.concatenate([held_k[i], kn[at:at + n][path]]), np.concatenate([held_v[i], vn[at:at + n][path]])
                length[i] += len(path)
            at += n
            places = np.arange(length[i])
            if window:
                places = places[(places < sinks) | (places > length[i] - window)]
            if places.size:
                slots = np.array(plan.table[i])[places // page] * page + places % page
                for g, a in zip(cache.read(slots), (held_k[i], held_v[i])):
                    stored = stored64(a, kind)[places]
                    within(g, stored, np.abs(stored) * (2.0 ** -11 + 2.0 ** -23) + 2.0 ** -25, f"rows of stream {i} after step {step}")
        assert np.isnan(got[n_new:]).all()
        assert dev.get(past, (streams,), np.int32).tolist() == length
    assert refused and again
    dev.check(dev.lib.mlvc_hip_graph_destroy(graph))
    dev.check(dev.lib.mlvc_hip_stream_destroy(stream))


# ------------------------------------------------------------ drafts that do not count

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("q_heads,heads,dim", [(4, 2, 64), (12, 1, 128), (40, 2, 64), (4, 2, 96), (2, 1, 264)])
@pytest.mark.parametrize("window", [0, 3, 40])
def test_drafts_past_longest_q_are_not_seen(dev, rng, kind, q_heads, heads, dim, window):
    """Masks that are no tree, with bits of drafts at longest_q and behind it: these add neither keys nor depth."""
    counts, lengths, longest_q = [9, 70, 3, 5], [60, 100, 41, 5], 3
    ctx = Contexts(dev, rng, Cache, kind, heads, dim, 16, lengths)
    masks = [0b010000001, 0b111, 0b101100100, 1 << 7, ALL, ALL] + [ALL] * (sum(counts) - 6)
    q = normal(rng, sum(counts), q_heads, dim)
    got = Drafts(ctx.cache, q, counts, masks, ctx.table, lengths, dim ** -0.5, window, 2, longest_q=longest_q).run()
    at = 0
    for i, (count, n) in enumerate(zip(counts, lengths)):
        past, here = n - count, [m & (1 << min(count, longest_q)) - 1 for m in masks[at:at + min(count, longest_q)]]
        depth = depths(here, longest_q)
        seen = np.zeros((len(here), n), bool)
        for r, m in enumerate(here):
            place = past + depth[r]
            for j in range(n):
                d = j - past
                if d < 0:
                    seen[r, j] = not window or place - j < window or j < 2
                elif d < len(here):
                    seen[r, j] = m >> d & 1 and (not window or depth[r] - depth[d] < window or past + depth[d] < 2)
        done = len(here)
        check(got[at:at + done], q[at:at + done], ctx.k[i], ctx.v[i], kind, dim ** -0.5, seen, f"stream {i}")
        assert np.isnan(got[at + done:at + count]).all()
        at += count


# ------------------------------------------------------------ the largest scores

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("q_heads,drafts,dim", [(2, 3, 64), (4, 8, 128), (6, 40, 128), (4, 64, 64), (3, 9, 96), (2, 40, 256), (2, 9, 512)])
@pytest.mark.parametrize("power", [8, 10, 11, 12, 13, 14])
def test_drafts_of_small_values_at_large_scores(dev, rng, kind, q_heads, drafts, dim, power):
    """Scores of 2^24 to 2^30, one key far above the others, on rows of V that are zero or far smaller than the others'.

    The best keys weigh 1 / count each and the others nothing (scores are 2^16 apart and more), so the result is the
    best rows' mean: a weight times its row's scale is rounded to FP16 (2^-11 of it, the scales 2^-16 are exact; scales
    below 2^-30 may be lost, with values up to 2^-24), the output once more."""
    n = 260
    level = {KV_E4M3: 448.0, KV_INT8: 127.0}.get(kind, 127.0)
    ctx = Contexts(dev, rng, Cache, kind, 1, dim, 16, [n])
    k = np.zeros((n, 1, dim), np.float16)
    k[:, 0, 0] = rng.permutation(n) + 1
    k[:, 0, 1] = n
    q = np.zeros((drafts, q_heads, dim), np.float16)
    q[..., 0] = 256 - np.arange(q_heads)
    masks, sk = tree(rng, drafts), stored64(k, kind)
    seen = drafts_seen(n, masks, 0, 0)
    order = np.argsort(k[:, 0, 0].astype(np.float64))
    for small in (0.0, 2.0 ** -24, level * 2.0 ** -16):
        v = ctx.v[0].copy()
        v[order[n // 2:]] = np.sign(v[order[n // 2:]]) * np.float16(small)
        ctx.cache.write(k, v, ctx.slots(0, np.arange(n)))
        got = Drafts(ctx.cache, q, [drafts], masks, ctx.table, [n], 2.0 ** power).run()
        sv = stored64(v, kind)
        for i in range(drafts):
            see = np.flatnonzero(seen[i])
            best = see[sk[see, 0, 0] == sk[see, 0, 0].max()]
            tol = np.abs(sv[best, 0]).max(0) * 2.0 ** -9 + 2.0 ** -23
            for h in range(q_heads):
                within(got[i, h], sv[best, 0].mean(0), tol, f"draft {i}, values of {small}")


# ------------------------------------------------------------ the last lengths

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("q_heads,dim,most,longest,window,sinks", [
    (4, 64, 4, (1 << 31) - 1, 50, 20),      # whole contexts: 16 rows, 64, padded, value by value
    (4, 128, 30, (1 << 31) - 1, 300, 0),
    (2, 96, 9, (1 << 31) - 1, 50, 20),
    (2, 264, 3, (1 << 31) - 1, 50, 20),
    (4, 64, 4, (1 << 31) - 1, 2500, 70),    # cut over workgroups
    (4, 128, 40, (1 << 31) - 1, 2500, 70),
    (2, 96, 9, (1 << 31) - 1, 2500, 70),
    (2, 264, 3, (1 << 31) - 1, 2100, 7),
    (4, 64, 4, (1 << 31) - 40, 300, 20),    # a cut before the last of them
])
def test_drafts_of_lengths_at_31_bits(dev, rng, kind, q_heads, dim, most, longest, window, sinks):
    """Contexts that end at 2^31 - 1 and a little before it, on pages of 2^16 tokens; what the window does not reach is on no page."""
    last, page, width = (1 << 31) - 1, 1 << 16, 1 << 15
    lengths, counts = [last, last - 20, 300, last - 31, last - 32, last - 1000], [most, 1, 2, 3, most, 2]
    cache = Cache(dev, kind, 3, page, 1, dim)
    table = np.full((len(lengths), width), -1, np.int32)
    table[:, 0], table[:, -1] = 1, 2        # sinks and the last tokens, the same for all streams
    k, v = normal(rng, 4096, 1, dim), normal(rng, 4096, 1, dim)
    at_end = np.arange(last - 4000, last)   # places of rows 96 ..
    cache.write(k[:96], v[:96], page + np.arange(96))
    cache.write(k[96:], v[96:], 2 * page + at_end % page)
    table[2, 0] = 2                         # the short one: the first rows of the last page's end, none of its window
    q = normal(rng, sum(counts), q_heads, dim)
    trees = [tree(rng, n) for n in counts]
    d = Drafts(cache, q, counts, [m for t in trees for m in t], table, lengths, dim ** -0.5, window, sinks, longest=longest)
    got, at = d.run(), 0
    for i, (count, n) in enumerate(zip(counts, lengths)):
        if i == 2:                          # rows that were never written
            at += count
            continue
        past, depth = n - count, depths(trees[i], count)
        places = np.concatenate([np.arange(sinks), np.arange(max(n - window - 100, last - 4000), min(n, longest))])
        rows = np.concatenate([np.arange(sinks), places[sinks:] - (last - 4000) + 96])
        seen = np.zeros((count, len(places)), bool)
        for r in range(count):
            place = past + depth[r]
            e = places - past
            other = past + np.array(depth)[np.clip(e, 0, count - 1)]
            at_place = np.where(e >= 0, other, places)
            mask = np.array([trees[i][r] >> b & 1 for b in range(count)], bool)[np.clip(e, 0, count - 1)]
            seen[r] = ((e < 0) | mask) & ((place - at_place < window) | (at_place < sinks))
        check(got[at:at + count], q[at:at + count], k[rows], v[rows], kind, dim ** -0.5, seen, f"stream {i}")
        at += count


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("behind", [0, 30, 63, 64, 200])
def test_window_of_keys_at_31_bits(dev, rng, causal, behind):
    """A sequence of 2^31 - 1 keys and a little fewer, of which the window sees the last and the sinks the first."""
    dim, n, tail, window, sinks = 1, (1 << 31) - 1 - behind, 1000, 100, 3
    base = dev.alloc(2 * ((1 << 31) + 8))
    rows = normal(rng, tail, 1, dim)
    for at, part in ((0, rows[:sinks]), (n - tail + sinks, rows[sinks:])):
        part = np.ascontiguousarray(part)
        dev.check(dev.lib.mlvc_hip_memcpy_h2d(base.value + 2 * at, part.ctypes.data, part.nbytes, None))
    q = normal(rng, 3, 2, dim)
    p = Prompt(dev, q, rows, rows, [3], [n], causal, 0.5)
    p.desc.k = p.desc.v = base.value
    p.desc.k_tokens = n
    seen = window_seen(3, tail, causal, window, sinks)
    want, tol = masked64(f64(q), f64(rows), f64(rows), 0.5, seen)
    within(Window(p, window, sinks).run(), want, tol)
