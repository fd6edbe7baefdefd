"""The operators that decode several tokens a step (page plans, attention under
a window, attention of drafts, kept drafts) against their definitions, through
the device C ABI."""

import ctypes as C

import numpy as np
import pytest

import mlvc_hip
from devmem import Dev
from drafts import ALL, Contexts, Drafts, Plan, Window, drafts_seen, keep, masked64, tops_of, tree, window_seen
from mlvc_hip import KV_E4M3, KV_F16, KV_INT8
from tokens import Cache, Padded, Prompt, Token, f64, stored64, within

pytestmark = pytest.mark.gpu

KINDS = [KV_F16, KV_E4M3, KV_INT8]


@pytest.fixture
def dev():
    d = Dev()
    yield d
    d.close()


def normal(rng, *shape):
    return rng.standard_normal(shape).astype(np.float16)


# ------------------------------------------------------------ plan

@pytest.mark.parametrize("streams,page,width,window,sinks,most", [
    (1, 16, 12, 0, 0, 40), (3, 48, 6, 0, 0, 64), (7, 16, 20, 50, 5, 33), (64, 16, 9, 1, 0, 7), (65, 32, 12, 100, 40, 64),
    (130, 16, 30, 33, 17, 64), (1024, 16, 4, 16, 1, 9), (1025, 16, 4, 0, 0, 9), (2500, 16, 6, 20, 16, 20),
])
def test_plan_steps(dev, rng, streams, page, width, window, sinks, most):
    """Steps of streams that keep some of their drafts, end and begin again."""
    plan = Plan(dev, streams, streams * width, page, width, window, sinks, rng.permutation(streams * width))
    length = np.zeros(streams, int)
    for step in range(6):
        room = width * page - length
        fresh = np.minimum(rng.integers(0, most + 1, streams), room)
        fresh[(room < page) | (rng.random(streams) < 0.05)] = -1
        masks = np.array([m for f in fresh if f > 0 for m in tree(rng, f)] or [0], np.uint64)
        total = int(fresh.clip(0).sum())
        masks = np.resize(masks, total + 3)
        past = length.copy()
        past[fresh < 0] = rng.integers(0, 1000)  # means nothing
        want = plan.step(past.tolist(), fresh.tolist(), total + (step % 3), masks if step % 2 else None)
        assert want["lacking"] == 0
        length = np.where(fresh < 0, 0, length + (fresh * rng.random(streams)).round().astype(int).clip(0))


def test_plan_again_gives_the_same(dev, rng):
    plan = Plan(dev, 9, 90, 16, 10, 40, 20, rng.permutation(90))
    plan.step([0] * 9, [100, 0, 17, 64, 1, 160, 3, 16, 15])
    args = [90, 0, 17, 60, 1, 100, 1, 16, 2], [5, 33, 1, 64, 0, 16, -1, 17, 64]
    first = plan.step(*args)
    first = {k: list(v) if isinstance(v, list) else v for k, v in first.items()}
    table = [list(r) for r in first["table"]]
    second = plan.step(*args)
    assert second["table"] == table and second["slots"] == first["slots"] and second["free"] == first["free"]


def test_plan_without_enough_pages(dev, rng):
    plan = Plan(dev, 6, 10, 16, 8, order=rng.permutation(10))
    want = plan.step([0] * 6, [40, 33, 0, 70, 1, 0])  # 3 + 3 pages; 5 are not there, and then 1 goes without too
    assert want["lacking"] == 2 and want["lengths"] == [40, 33, 0, 0, 0, 0] and len(want["free"]) == 4
    want = plan.step([40, 33, 0, 0, 0, 0], [8, 15, 0, -1, 1, 0])  # what is held suffices for the first two
    assert want["lacking"] == 0 and len(want["free"]) == 3
    want = plan.step([48, 48, 0, 0, 1, 0], [200, 1, 1, 0, 1, 1])  # beyond its row: the others go on
    assert want["lacking"] == 1 and want["lengths"] == [48, 49, 1, 0, 2, 1]


def test_plan_cut_rows_and_no_positions(dev, rng):
    plan = Plan(dev, 3, 30, 16, 10, order=rng.permutation(30))
    plan.step([0, 0, 0], [20, 30, 7], tokens=41)                   # rows end inside the second stream
    plan.step([20, 30, 7], [1, 1, 1], tokens=9, positions=False)   # padding rows
    plan.step([21, 31, 8], [0, 0, 0], tokens=0)
    none = Plan(dev, 0, 4, 16, 3)
    none.step([], [], tokens=5)
    flat = Plan(dev, 2, 0, 16, 0)
    assert flat.step([0, 0], [1, 0])["lacking"] == 1


def test_plan_of_a_long_prompt(dev, rng):
    plan = Plan(dev, 5, 1500, 16, 700, 500, 4, rng.permutation(1500))
    plan.step([0] * 5, [8160, 1, 5000, 0, 3001])
    plan.step([8160, 1, 5000, 0, 3001], [1, 2000, 8, 600, -1])


def test_plan_of_lengths_at_31_bits(dev):
    page, last = 1 << 28, (1 << 31) - 1
    plan = Plan(dev, 1, 7, page, 9, window=16)
    get = lambda at, n: dev.get(at, (n,), np.int32).tolist()  # noqa: E731

    def step(past, fresh, tokens=8):
        mlvc_hip.kv_plan(plan.desc([past], [fresh], tokens))
        return get(plan.d_lengths, 1)[0], get(plan.d_lacking, 1)[0], get(plan.slots, tokens)

    assert step(0, 1 << 30)[:2] == (1 << 30, 0)
    assert step(1 << 30, (1 << 30) - 5)[:2] == (last - 4, 0)
    page_of = get(plan.d_table, 9)[7] * page
    assert get(plan.d_table, 9)[8] == -1 and page_of >= 0
    # One more than a length can count: the row has an entry for it, and it goes without.
    assert step(last - 4, 5) == (last - 4, 1, [-1] * 8)
    assert step(last - 4, 4) == (last, 0, [page_of + page - 5 + i for i in range(4)] + [-1] * 4)


# ------------------------------------------------------------ kept drafts

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,dim,page", [(2, 64, 16), (3, 128, 48), (1, 24, 16), (5, 96, 32), (2, 512, 16), (9, 8, 64)])
def test_keep(dev, rng, kind, heads, dim, page):
    counts = [8, 1, 64, 0, 5, 33, 6]
    lengths = [8, 40, 64 + 13, 9, 5, 33 + 31, 6 + 16]
    kept = np.full((7, 64), -1)
    kept[0, :4] = [0, 3, 4, 7]
    kept[1, :1] = [0]
    kept[2] = rng.permutation(64)               # every row moves
    kept[3, :2] = [0, 1]                        # no drafts: nothing is kept
    kept[4, :6] = [4, 4, 0, 5, 1, 2]            # twice the same, then one that is not there
    kept[5, :5] = [1, 2, 3, 4, 32]              # each into the place of the one before
    ctx = Contexts(dev, rng, Cache, kind, heads, dim, page, lengths)
    new = keep(ctx.cache, ctx.table, counts, lengths, kept)
    for i, (count, n) in enumerate(zip(counts, lengths)):
        path = []
        for d in kept[i]:
            if not 0 <= d < count:
                break
            path.append(d)
        assert new[i] == n - count + len(path)
        order = np.arange(n)
        order[n - count:n - count + len(path)] = n - count + np.array(path, int)
        if n == 0:
            continue
        got = ctx.cache.read(ctx.slots(i, np.arange(n)))
        for g, x in zip(got, (ctx.k[i], ctx.v[i])):
            want = stored64(x, kind)[order]
            within(g, want, np.abs(want) * (2.0 ** -11 + 2.0 ** -23) + 2.0 ** -25)


def test_keep_of_rows_that_are_not_there(dev, rng):
    ctx = Contexts(dev, rng, Cache, KV_INT8, 2, 64, 16, [40, 40, 3])
    before = [ctx.cache.read(ctx.slots(i, np.arange(n))) for i, n in enumerate((40, 40, 3))]
    table = ctx.table.copy()
    table[1, 2] = -1                 # places 32 to 47 of the second are gone
    table[0, 1] = 10 ** 6            # places 16 to 31 of the first are not in the cache
    new = keep(ctx.cache, table, [30, 10, 8], [40, 40, 3], [[7, 25], [0, 3], [6, 7]])
    assert new == [12, 32, 0]        # the third says that it has more drafts than tokens
    # First: its context ends at 10; draft 7 is at place 17, on the page that is not there; draft 25 at 35 moves to 11.
    for g, b in zip(ctx.cache.read(ctx.slots(0, np.arange(40))), before[0]):
        want = b.copy()
        want[11] = b[35]
        assert np.array_equal(g.view(np.uint16), want.view(np.uint16))
    # Second: 30 stays, 33 is not there.
    for g, b in zip(ctx.cache.read(ctx.slots(1, np.arange(40))), before[1]):
        assert np.array_equal(g.view(np.uint16), b.view(np.uint16))
    # Third: its drafts begin five places before the cache does: draft 6 (place 1) has nowhere to go.
    for g, b in zip(ctx.cache.read(ctx.slots(2, np.arange(3))), before[2]):
        assert np.array_equal(g.view(np.uint16), b.view(np.uint16))


def test_keep_past_32_bits(dev, rng):
    """A cache of 5 GB of keys."""
    pages, page, heads, dim = 40000, 16, 64, 128
    desc = mlvc_hip.KvCache(kind=KV_INT8, pages=pages, page_size=page, heads=heads, head_dim=dim)
    nbytes, scales = mlvc_hip.kv_cache_bytes(desc)
    desc.k, desc.v, desc.k_scale, desc.v_scale = dev.alloc(nbytes), dev.alloc(nbytes), dev.alloc(scales), dev.alloc(scales)
    cache = Cache.__new__(Cache)
    cache.dev, cache.kind, cache.page_size, cache.heads, cache.dim, cache.pages, cache.desc = dev, KV_INT8, page, heads, dim, pages, desc
    table = np.array([[17, 39999, 33333]])
    places = np.arange(48)
    slots = table[0, places // page] * page + places % page
    k, v, q = normal(rng, 48, heads, dim), normal(rng, 48, heads, dim), normal(rng, 2, heads, dim)
    cache.write(k, v, slots)
    got = Drafts(cache, q, [2], None, table, [48], 0.09).run()
    sk, sv = stored64(k, KV_INT8), stored64(v, KV_INT8)
    want, tol = masked64(f64(q), sk, sv, 0.09, drafts_seen(48, [1, 3], 0, 0), tops_of(v, KV_INT8))
    within(got, want, tol)
    assert keep(cache, table, [20], [48], [[3, 19]]) == [30]
    order = np.arange(48)
    order[28:30] = [31, 47]
    for g, x in zip(cache.read(slots), (sk, sv)):
        within(g, x[order], np.abs(x[order]) * (2.0 ** -11 + 2.0 ** -23) + 2.0 ** -25)


# ------------------------------------------------------------ attention under a window

def _window(dev, rng, queries, keys, q_heads, kv_heads, dim, causal, window, sinks, extra=0, shift=0, spread=1.0):
    q = normal(rng, sum(queries), q_heads, dim) * np.float16(spread)
    k, v = (normal(rng, sum(keys), kv_heads, dim) for _ in range(2))
    got = Window(Prompt(dev, q, k, v, queries, keys, causal, dim ** -0.5, extra, shift), window, sinks).run()
    i = j = 0
    for nq, nk in zip(queries, keys):
        want, tol = masked64(f64(q[i:i + nq]), f64(k[j:j + nk]), f64(v[j:j + nk]), dim ** -0.5, window_seen(nq, nk, causal, window, sinks))
        within(got[i:i + nq], want, tol, f"sequence of {nq} on {nk}")
        i, j = i + nq, j + nk


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (31, 0), (32, 33), (64, 4), (100, 130), (129, 0), (1000, 5)])
@pytest.mark.parametrize("queries,keys", [
    ([1], [1]), ([33], [33]), ([257], [257]), ([1, 240, 0, 65, 3], [1, 240, 7, 65, 3]),
    ([1, 17, 130], [300, 64, 260]),      # behind what came before
    ([40, 200, 5], [7, 64, 0]),          # more queries than keys: rows that see nothing
])
def test_window_lengths(dev, rng, queries, keys, window, sinks, dim, causal):
    _window(dev, rng, queries, keys, 2, 1, dim, causal, window, sinks)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim,q_heads,kv_heads,extra,shift", [
    (64, 4, 4, 0, 0), (128, 8, 1, 0, 0), (64, 6, 2, 64, 0), (128, 16, 1, 8, 16),
    (64, 3, 1, 1, 0), (128, 2, 2, 0, 1),                       # off 16 bytes
    (96, 3, 1, 0, 0), (33, 2, 1, 0, 0), (512, 1, 1, 0, 0),     # other heads
    (8, 4, 2, 0, 0), (40, 6, 3, 8, 8), (120, 4, 2, 0, 0), (136, 4, 4, 0, 0), (200, 4, 2, 64, 0), (256, 2, 2, 0, 8), (264, 2, 1, 0, 0),
    (96, 2, 2, 1, 0), (256, 2, 2, 0, 1),
])
def test_window_heads_and_strides(dev, rng, dim, q_heads, kv_heads, extra, shift, causal):
    _window(dev, rng, [70, 9], [200, 9], q_heads, kv_heads, dim, causal, 40, 6, extra, shift)


@pytest.mark.parametrize("queries,keys,q_heads,dim,causal,window,sinks", [
    ([240], [240], 16, 64, True, 80, 4), ([700, 600], [700, 600], 16, 64, False, 100, 0), ([1500], [1500], 16, 64, True, 333, 70),
    ([10], [1500], 16, 64, True, 700, 4), ([10], [1500], 16, 128, False, 1, 300), ([920], [920], 16, 128, True, 500, 1),
    ([2040], [2040], 16, 128, True, 129, 64), ([1, 1200, 333, 64, 700], [1, 1300, 333, 900, 700], 16, 128, True, 256, 9),
    ([3000, 700], [3000, 900], 16, 64, True, 64, 130), ([4097], [4097], 16, 128, True, 640, 0), ([1100, 40], [1100, 2000], 5, 64, False, 65, 65),
    ([30] * 70, [100] * 70, 3, 64, True, 33, 2), ([200] * 66, [230] * 66, 2, 128, False, 50, 3),
])
def test_window_tiles(dev, rng, queries, keys, q_heads, dim, causal, window, sinks):
    """Every shape of workgroup, windows that begin and end inside tiles, tiles of sinks beside them."""
    _window(dev, rng, queries, keys, q_heads, 1, dim, causal, window, sinks)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [24, 96, 160, 256])
@pytest.mark.parametrize("queries,keys,q_heads,window,sinks", [
    ([1, 240, 0, 65, 3], [1, 240, 7, 65, 3], 4, 33, 4), ([1, 17, 130], [300, 64, 260], 4, 100, 130), ([40, 200, 5], [7, 64, 0], 4, 1, 0),
    ([1500], [1500], 16, 333, 70), ([1100, 40], [1100, 2000], 16, 65, 65), ([30] * 70, [100] * 70, 6, 33, 2),
    ([300, 20], [300, 50], 4, 5000, 9),                        # wider than all there is
])
def test_window_padded_heads(dev, rng, queries, keys, q_heads, dim, causal, window, sinks):
    _window(dev, rng, queries, keys, q_heads, 2, dim, causal, window, sinks)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("queries,keys,q_heads,dim,window,sinks", [
    ([70], [70], 2, 64, 20, 3), ([200, 33], [300, 33], 2, 128, 40, 70), ([900], [900], 16, 64, 31, 5), ([520], [700], 16, 128, 300, 0),
    ([300], [300], 2, 96, 33, 2), ([1200], [1200], 16, 128, 1, 66), ([400], [500], 3, 264, 33, 2),
    ([1200], [1200], 16, 72, 40, 66), ([500, 90], [500, 300], 3, 184, 33, 5), ([700], [700], 2, 256, 100, 3),
])
def test_window_of_infinite_values(dev, rng, queries, keys, q_heads, dim, window, sinks, causal):
    """Infinities and NaN among the values reach the queries that see them, and no others."""
    q, k, v = normal(rng, sum(queries), q_heads, dim), normal(rng, sum(keys), 1, dim), normal(rng, sum(keys), 1, dim)
    for value in (np.inf, -np.inf, np.nan):
        for _ in range(max(2, sum(keys) // 60)):
            v[rng.integers(0, sum(keys)), 0, rng.integers(0, dim)] = value
    v[0, 0, 1], v[min(sinks, 60), 0, 2] = np.inf, -np.inf
    got = Window(Prompt(dev, q, k, v, queries, keys, causal, dim ** -0.5), window, sinks).run()
    i = j = 0
    for nq, nk in zip(queries, keys):
        want, tol = masked64(f64(q[i:i + nq]), f64(k[j:j + nk]), f64(v[j:j + nk]), dim ** -0.5, window_seen(nq, nk, causal, window, sinks))
        assert np.array_equal(np.isnan(got[i:i + nq]), np.isnan(want)) and np.array_equal(np.isinf(got[i:i + nq]), np.isinf(want))
        inf = np.isinf(want)
        assert np.array_equal(got[i:i + nq][inf] > 0, want[inf] > 0)
        within(got[i:i + nq], want, tol)
        i, j = i + nq, j + nk


@pytest.mark.parametrize("dim", [64, 128, 80, 232])
def test_window_peaked_and_small_weights(dev, rng, dim):
    """Scores far apart, and many small weights beside a large one among the sinks."""
    for spread in (20.0, 0.01):
        _window(dev, rng, [300], [500], 2, 1, dim, True, 200, 40, spread=spread)
    n = 1500
    q, k, v = np.zeros((3, 1, dim), np.float16), np.zeros((n, 1, dim), np.float16), normal(rng, n, 1, dim)
    q[..., 0], k[0, 0, 0] = 1, 16           # the first key weighs e^16 times the others
    v[0] = 0
    got = Window(Prompt(dev, q, k, v, [3], [n], True, 1.0), 1200, 1).run()
    want, tol = masked64(f64(q), f64(k), f64(v), 1.0, window_seen(3, n, True, 1200, 1))
    within(got, want, tol)


def test_window_strides_past_32_bits(dev, rng):
    """Keys 2^31 halves and more from the first."""
    dim, n, stride = 64, 40, 1 << 26
    base = dev.alloc(2 * (n * stride + dim))
    rows = normal(rng, n, 1, dim)
    for i in range(n):
        dev.check(dev.lib.mlvc_hip_memcpy_h2d(base.value + 2 * i * stride, rows[i].ctypes.data, 2 * dim, None))
    q = normal(rng, n, 1, dim)
    p = Prompt(dev, q, rows, rows, [n], [n], True, 0.125)
    p.desc.k = p.desc.v = base.value
    p.desc.k_stride = p.desc.v_stride = stride
    want, tol = masked64(f64(q), f64(rows), f64(rows), 0.125, window_seen(n, n, True, 9, 2))
    within(Window(p, 9, 2).run(), want, tol)


@pytest.mark.parametrize("dim", [64, 128, 40])
@pytest.mark.parametrize("causal", [False, True])
def test_window_of_all_sinks_is_the_prompt(dev, rng, dim, causal):
    """Sinks that reach to the last key."""
    q, k, v = normal(rng, 150, 2, dim), normal(rng, 200, 1, dim), normal(rng, 200, 1, dim)
    p = Prompt(dev, q, k, v, [150], [200], causal, 0.1)
    for sinks in (200, 2 ** 31 - 1):
        want, tol = masked64(f64(q), f64(k), f64(v), 0.1, window_seen(150, 200, causal, 0, 0))
        within(Window(p, 1, sinks).run(), want, tol)


def test_window_of_none_is_the_prompt(dev, rng):
    q, k, v = (normal(rng, 300, 2, 64) for _ in range(3))
    for causal in (False, True):
        p = Prompt(dev, q, k, v, [200, 100], [200, 100], causal, 0.125)
        want = p.run()
        for window in (0, 600, 2 ** 31 - 1):
            got = Window(p, window, 7).run()
            assert np.array_equal(got.view(np.uint16), want.view(np.uint16))


# ------------------------------------------------------------ attention of drafts

def _drafts(dev, rng, kind, q_heads, heads, dim, page, counts, lengths, window=0, sinks=0, extra=0, shift=0, chain=False, spread=1.0):
    ctx = Contexts(dev, rng, Cache, kind, heads, dim, page, lengths, spread)
    q = normal(rng, sum(counts), q_heads, dim)
    trees = [[(2 << i) - 1 for i in range(n)] if chain else tree(rng, n) for n in counts]
    masks = None if chain else [m for t in trees for m in t] + [0]
    got = Drafts(ctx.cache, q, counts, masks, ctx.table, lengths, dim ** -0.5, window, sinks, extra=extra, shift=shift).run()
    at = 0
    for i, (count, n) in enumerate(zip(counts, lengths)):
        want, tol = masked64(f64(q[at:at + count]), stored64(ctx.k[i], kind), stored64(ctx.v[i], kind), dim ** -0.5,
                             drafts_seen(n, trees[i], window, sinks), tops_of(ctx.v[i], kind))
        within(got[at:at + count], want, tol, f"stream {i}: {count} drafts in {n} tokens")
        at += count


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (3, 2), (50, 0), (64, 70), (300, 4)])
@pytest.mark.parametrize("q_heads,heads,dim,page", [(8, 2, 64, 16), (4, 1, 128, 48)])
def test_drafts(dev, rng, kind, q_heads, heads, dim, page, window, sinks):
    _drafts(dev, rng, kind, q_heads, heads, dim, page, [1, 5, 0, 64, 2, 16, 33, 1], [1, 5, 9, 64 + 17, 700, 333, 100, 640], window, sinks)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("q_heads,heads,dim,page,extra,shift", [
    (16, 1, 64, 64, 0, 0), (40, 2, 64, 32, 0, 0), (3, 3, 128, 16, 64, 8), (5, 1, 128, 32, 0, 0), (12, 4, 64, 48, 0, 0),
    (4, 2, 64, 16, 1, 0), (2, 2, 128, 16, 0, 3),                 # off 16 bytes
    (4, 2, 96, 16, 0, 0), (2, 1, 24, 32, 0, 0), (1, 1, 512, 16, 0, 0),
])
def test_drafts_heads_and_strides(dev, rng, kind, q_heads, heads, dim, page, extra, shift):
    _drafts(dev, rng, kind, q_heads, heads, dim, page, [7, 1, 20], [190, 33, 20], 60, 9, extra, shift)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (400, 20)])
def test_drafts_in_a_chain_on_long_contexts(dev, rng, kind, dim, window, sinks):
    """A chain of drafts, contexts that are cut over workgroups."""
    _drafts(dev, rng, kind, 4, 2, dim, 32, [3, 1, 9], [2100, 1500, 30], window, sinks, chain=True)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_heads,heads,counts,lengths,window,sinks", [
    # Whole contexts: 16 rows of many streams, 32 rows, 64, 128.
    (4, 2, [1, 3, 2] * 50, [5, 300, 77] * 50, 0, 0),
    (4, 1, [8, 5, 6] * 35, [205, 70, 33] * 35, 64, 40),
    (16, 8, [20, 17, 1] * 11, [150, 64, 40] * 11, 0, 0),
    (16, 8, [64, 40, 33, 50, 1] * 13, [70, 130, 64, 96, 33] * 13, 50, 3),
    # Cut ones: 32 rows, 64, 64 of many streams, 128.
    (4, 2, [15, 9] * 20, [2600, 31] + [77, 40] * 19, 0, 0),
    (6, 2, [20, 16] * 20, [2600, 31] + [77, 40] * 19, 0, 0),
    (16, 8, [20] * 33, [2300] + [60] * 31 + [2100], 0, 0),
    (4, 2, [64, 3, 33], [8300, 40, 700], 0, 0),
    (4, 2, [64, 3, 33], [9000, 40, 8700], 8400, 100),
])
def test_drafts_shapes(dev, rng, kind, dim, q_heads, heads, counts, lengths, window, sinks):
    """Every number of rows a workgroup takes, contexts whole and cut."""
    _drafts(dev, rng, kind, q_heads, heads, dim, 16, counts, lengths, window, sinks)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("q_heads,heads,dim,extra,shift", [(4, 2, 96, 0, 0), (3, 1, 24, 0, 0), (2, 1, 200, 0, 0), (2, 1, 264, 0, 0), (4, 2, 64, 1, 0), (2, 1, 128, 0, 3)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1500, 40)])
def test_drafts_cut_other_heads(dev, rng, kind, q_heads, heads, dim, extra, shift, window, sinks):
    """Contexts that are cut, heads and rows of the plain kernel and of the padded ones."""
    _drafts(dev, rng, kind, q_heads, heads, dim, 16, [5, 1, 9, 0], [2100, 40, 1700, 3], window, sinks, extra, shift)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [16, 96, 144, 256])
@pytest.mark.parametrize("q_heads,heads,counts,lengths,window,sinks", [
    (4, 2, [1, 3, 2, 0, 9], [5, 300, 77, 30, 8], 0, 0),                # whole contexts, few rows
    (16, 8, [64, 40, 33, 50, 1] * 5, [70, 130, 64, 96, 33] * 5, 50, 3),  # rows of two workgroups
    (6, 2, [20, 16] * 20, [2600, 31] + [77, 40] * 19, 0, 0),           # cut
    (4, 2, [64, 3, 33], [5000, 40, 4700], 4400, 100),
])
def test_drafts_padded_heads(dev, rng, kind, dim, q_heads, heads, counts, lengths, window, sinks):
    _drafts(dev, rng, kind, q_heads, heads, dim, 16, counts, lengths, window, sinks)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_heads,drafts,n", [(2, 3, 700), (4, 16, 700), (6, 40, 300), (2, 5, 1500), (4, 60, 6000), (2, 20, 9000)])
def test_drafts_of_zero_values_and_far_scores(dev, rng, kind, dim, q_heads, drafts, n):
    """Zero rows of V that weigh most, rows of far smaller values beside large ones, scores far apart."""
    ctx = Contexts(dev, rng, Cache, kind, 1, dim, 16, [n])
    k, v = ctx.k[0], ctx.v[0]
    v[: n // 3] *= np.float16(2.0 ** -12)
    top = rng.permutation(n)[: n // 4]
    v[top] = 0
    k[top] *= np.float16(3)
    k[n // 2:] *= np.float16(8)
    ctx.cache.write(k, v, ctx.slots(0, np.arange(n)))
    q = normal(rng, drafts, q_heads, dim)
    masks = tree(rng, drafts)
    got = Drafts(ctx.cache, q, [drafts], masks, ctx.table, [n], 0.2).run()
    want, tol = masked64(f64(q), stored64(k, kind), stored64(v, kind), 0.2, drafts_seen(n, masks, 0, 0), tops_of(v, kind))
    within(got, want, tol)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("q_heads,drafts,dim", [(2, 3, 64), (4, 8, 128), (6, 40, 128), (4, 64, 64), (3, 9, 96), (2, 9, 512)])
def test_drafts_of_large_scores(dev, rng, kind, q_heads, drafts, dim):
    """Scores of 2^22 and more, whose last place is more than the weights' own: the largest decides."""
    n = 260
    ctx = Contexts(dev, rng, Cache, kind, 1, dim, 16, [n])
    k = np.zeros((n, 1, dim), np.float16)
    k[:, 0, 0] = rng.permutation(n) + 1     # whole multiples of a power of two once scaled: one key far above the others
    k[:, 0, 1] = n                          # the rows' largest value: quantised alike
    ctx.cache.write(k, ctx.v[0], ctx.slots(0, np.arange(n)))
    q = np.zeros((drafts, q_heads, dim), np.float16)
    q[..., 0] = 256
    masks = tree(rng, drafts)
    got = Drafts(ctx.cache, q, [drafts], masks, ctx.table, [n], 2.0 ** 18).run()
    sk, sv, seen = stored64(k, kind), stored64(ctx.v[0], kind), drafts_seen(n, masks, 0, 0)
    for i in range(drafts):
        see = np.flatnonzero(seen[i])
        best = see[sk[see, 0, 0] == sk[see, 0, 0].max()]
        want = sv[best, 0].mean(0)
        tol = np.abs(sv[best, 0]).max(0) * 2.0 ** -9 + 2.0 ** -24
        for h in range(q_heads):
            within(got[i, h], want, tol, f"draft {i}")


@pytest.mark.parametrize("q_heads,drafts,dim,n", [(2, 3, 64, 200), (4, 8, 128, 900), (6, 40, 128, 300), (4, 64, 64, 3000), (4, 30, 128, 5000), (2, 9, 96, 100), (2, 9, 96, 2000), (2, 40, 256, 3000), (2, 9, 264, 2000)])
def test_drafts_of_infinite_values(dev, rng, q_heads, drafts, dim, n):
    """Infinities and NaN among the values of an FP16 cache reach the drafts that see them, and no others."""
    ctx = Contexts(dev, rng, Cache, KV_F16, 1, dim, 16, [n, n])
    trees = [tree(rng, drafts), tree(rng, drafts)]
    for stream in range(2):
        v = ctx.v[stream]
        for value in (np.inf, -np.inf, np.nan):
            if stream == 0:
                v[rng.integers(0, n - drafts), 0, rng.integers(0, dim)] = value
            for _ in range(3):
                v[n - drafts + rng.integers(0, drafts), 0, rng.integers(0, dim)] = value
        ctx.cache.write(ctx.k[stream], v, ctx.slots(stream, np.arange(n)))
    q = normal(rng, 2 * drafts, q_heads, dim)
    for window in (0, 70):
        got = Drafts(ctx.cache, q, [drafts] * 2, trees[0] + trees[1], ctx.table, [n, n], 0.1, window, 3).run()
        for i in range(2):
            want, tol = masked64(f64(q[i * drafts:(i + 1) * drafts]), f64(ctx.k[i]), f64(ctx.v[i]), 0.1, drafts_seen(n, trees[i], window, 3))
            g = got[i * drafts:(i + 1) * drafts]
            assert np.array_equal(np.isnan(g), np.isnan(want)) and np.array_equal(np.isinf(g), np.isinf(want))
            inf = np.isinf(want)
            assert np.array_equal(g[inf] > 0, want[inf] > 0)
            within(g, want, tol)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128])
def test_one_draft_is_the_token_step(dev, rng, kind, dim):
    ctx = Contexts(dev, rng, Cache, kind, 2, dim, 16, [1, 500, 37, 1300])
    q = normal(rng, 4, 8, dim)
    a = Drafts(ctx.cache, q, [1] * 4, None, ctx.table, [1, 500, 37, 1300], 0.1).run().astype(np.float64)
    b = Token(ctx.cache, q, ctx.table, [1, 500, 37, 1300], 0.1).run().astype(np.float64)
    # Both are within their tolerances of the same number: one rounding of the output and one of the weights each.
    top = max(np.abs(f64(v)).max() for v in ctx.v)
    assert np.abs(a - b).max() <= top * (2.0 ** -10 + 2.0 ** -10)


@pytest.mark.parametrize("dim", [64, 96, 264])
def test_drafts_of_any_masks(dev, rng, dim):
    """Masks that are no tree: later drafts, none at all, bits past the last draft."""
    lengths = [6, 200]
    ctx = Contexts(dev, rng, Cache, KV_INT8, 2, dim, 16, lengths)
    masks = [[0, 1 << 5, 0b111111, ALL, 0b10, 1 << 40], [0, 0b1000, ALL, 1 << 63]]
    q = normal(rng, 10, 2, dim)
    got = Drafts(ctx.cache, q, [6, 4], masks[0] + masks[1], ctx.table, lengths, 0.1).run()
    at = 0
    for i, (n, m) in enumerate(zip(lengths, masks)):
        here = [x & (1 << len(m)) - 1 for x in m]
        want, tol = masked64(f64(q[at:at + len(m)]), stored64(ctx.k[i], KV_INT8), stored64(ctx.v[i], KV_INT8), 0.1,
                             drafts_seen(n, here, 0, 0), tops_of(ctx.v[i], KV_INT8))
        within(got[at:at + len(m)], want, tol)
        at += len(m)
    assert not got[0].any() and not got[5].any()  # nothing seen


@pytest.mark.parametrize("dim", [64, 128, 40, 96])
def test_drafts_rows_that_are_not_computed(dev, rng, dim):
    """More drafts than longest_q, than 64, than rows of q; more drafts than tokens; rows past the last stream."""
    counts, lengths = [70, 4, 9, 6], [100, 300, 5, 40]
    ctx = Contexts(dev, rng, Cache, KV_F16, 1, dim, 16, lengths)
    q = normal(rng, sum(counts) + 3, 2, dim)
    rows = sum(counts[:3]) + 2                      # the last stream's rows end after two
    trees = [tree(rng, min(n, 64)) for n in counts]
    trees[0] += [1 << 63] * 6                       # past the 64th draft
    masks = [m for t in trees for m in t]
    for longest_q in (64, 3):
        d = Drafts(ctx.cache, q, counts, masks + [0] * 3, ctx.table, lengths, 0.1, longest_q=longest_q)
        d.desc.q_tokens = rows
        got = d.run()
        at = 0
        for i, (count, n) in enumerate(zip(counts, lengths)):
            done = min(count, longest_q, rows - at)
            seen = np.zeros((done, n), bool)
            for r in range(done):
                for j in range(n):
                    e = j - (n - count)
                    seen[r, j] = e < 0 or (e < 64 and trees[i][r] >> e & 1)
            want, tol = masked64(f64(q[at:at + done]), f64(ctx.k[i]), f64(ctx.v[i]), 0.1, seen)
            within(got[at:at + done], want, tol, f"stream {i}")
            assert np.isnan(got[at + done:min(at + count, len(q))]).all()
            at += count


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 72, 160])
@pytest.mark.parametrize("window", [0, 40])
def test_drafts_unseen_places_do_not_reach(dev, rng, kind, dim, window):
    """NaN and infinities in drafts of other branches, behind the window, past the end and on pages outside."""
    lengths, counts = [150, 64, 37], [8, 3, 2]
    ctx = Contexts(dev, rng, Cache, kind, 2, dim, 16, lengths)
    trees = [[1, 3, 5, 11, 21, 1 << 5, 1 << 5 | 1 << 6, 3 | 1 << 7], [1, 3, 5], [1, 2]]
    bad = np.full((1, 2, dim), np.nan, np.float16)
    bad[..., ::2] = np.inf
    seen = [drafts_seen(n, t, window, 2) for n, t in zip(lengths, trees)]
    hidden = [[142 + 4], [63], [36]]                # drafts that few others see
    for i, places in enumerate(hidden):
        for p in places:
            ctx.cache.write(bad, bad, ctx.slots(i, [p]))
    if window:
        for p in range(5, 100, 7):
            ctx.cache.write(bad, bad, ctx.slots(0, [p]))
    past_end = [ctx.table[i, n // 16] * 16 + n % 16 for i, n in enumerate(lengths) if n % 16]
    ctx.cache.write(np.repeat(bad, len(past_end), 0), np.repeat(bad, len(past_end), 0), past_end)
    table = ctx.table.copy()
    table[0, 3] = -1
    seen[0][:, 48:64] = False
    table[1, 0] = 10 ** 6
    seen[1][:, :16] = False
    q = normal(rng, sum(counts), 4, dim)
    got = Drafts(ctx.cache, q, counts, [m for t in trees for m in t], table, lengths, 0.1, window, 2).run()
    at = 0
    for i, (count, n) in enumerate(zip(counts, lengths)):
        want, tol = masked64(f64(q[at:at + count]), stored64(ctx.k[i], kind), stored64(ctx.v[i], kind), 0.1, seen[i], tops_of(ctx.v[i], kind))
        clean = ~seen[i][:, hidden[i]].any(1)
        within(got[at:at + count][clean], want[clean], tol[clean], f"stream {i}")
        assert np.isnan(got[at:at + count][~clean]).all()  # those that see it
        at += count


@pytest.mark.parametrize("dim", [64, 128, 40, 96])
def test_drafts_of_the_widest_window(dev, rng, dim):
    """A window and sinks of 2^31 - 1, more drafts than tokens among the streams: nothing is cut."""
    counts, lengths = [5, 9, 20], [300, 4, 40]
    ctx = Contexts(dev, rng, Cache, KV_INT8, 1, dim, 16, lengths)
    q = normal(rng, sum(counts), 4, dim)
    masks = [m for n in counts for m in tree(rng, n)]
    got = [Drafts(ctx.cache, q, counts, masks, ctx.table, lengths, 0.1, *w).run().view(np.uint16)
           for w in ((0, 0), (2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1), (1, 2 ** 31 - 1))]
    for g in got[1:]:
        assert np.array_equal(g, got[0])


@pytest.mark.parametrize("kind", KINDS)
def test_drafts_are_repeatable(dev, rng, kind):
    ctx = Contexts(dev, rng, Cache, kind, 2, 64, 16, [2500, 700, 90])
    q = normal(rng, 24, 8, 64)
    d = Drafts(ctx.cache, q, [16, 7, 1], tree(rng, 16) + tree(rng, 7) + [1], ctx.table, [2500, 700, 90], 0.125)
    first = d.run().view(np.uint16)
    for _ in range(4):
        assert np.array_equal(d.run().view(np.uint16), first)


# ------------------------------------------------------------ together

@pytest.mark.parametrize("kind", KINDS)
def test_decode_with_drafts_captured(dev, rng, kind):
    """Plan, write, attend to and keep drafts, captured once and replayed, against the definition: contexts
    with a window whose old pages go back to the pool."""
    streams, heads, q_heads, dim, page, window, sinks, most = 3, 2, 4, 64, 16, 40, 5, 8
    width = 40
    plan = Plan(dev, streams, streams * 9, page, width, window, sinks, rng.permutation(streams * 9))
    cache = Cache(dev, kind, streams * 9, page, heads, dim)
    put = lambda shape, t: dev.put(np.zeros(shape, t))  # noqa: E731
    tokens = streams * most
    past, fresh, kept, seen = put(streams, np.int32), put(streams, np.int32), put((streams, most), np.int32), put(tokens, np.uint64)
    x = np.zeros((tokens, heads, dim), np.float16)
    q, k, v = Padded(dev, np.zeros((tokens, q_heads, dim), np.float16)), Padded(dev, x), Padded(dev, x)
    out = Padded(dev, np.full((tokens, q_heads, dim), np.nan, np.float16))
    pd = plan.desc(past, fresh, tokens, seen)
    rows = mlvc_hip.KvRows(tokens=tokens, k=k.at, v=v.at, k_stride=k.stride, v_stride=v.stride, slots=plan.slots)
    ad = mlvc_hip.DraftAttention(cache=C.pointer(cache.desc), streams=streams, q_heads=q_heads, q_tokens=tokens, longest_q=most,
                                 q=q.at, out=out.at, q_stride=q.stride, out_stride=out.stride, starts=plan.d_starts, seen=seen,
                                 table=plan.d_table, table_stride=width, lengths=plan.d_lengths, longest=width * page,
                                 window=window, sinks=sinks, scale=0.125)
    ad.workspace_bytes = mlvc_hip.attention_drafts_workspace_bytes(ad)
    if ad.workspace_bytes:
        ad.workspace = dev.put(np.full(ad.workspace_bytes, 0xFF, np.uint8))
    kd = mlvc_hip.KvKeep(cache=C.pointer(cache.desc), streams=streams, table=plan.d_table, table_stride=width, starts=plan.d_starts,
                         lengths=plan.d_lengths, kept=kept, kept_stride=most, lengths_out=past)
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

    length = [0] * streams
    held_k, held_v = [np.zeros((0, heads, dim), np.float16) for _ in range(streams)], [np.zeros((0, heads, dim), np.float16) for _ in range(streams)]
    for step in range(14):
        counts = [int(rng.integers(1, most + 1)) for _ in range(streams)]
        if step == 6:
            counts[1], length[1] = -1, 0
            held_k[1] = held_v[1] = held_k[1][:0]
        trees = [tree(rng, max(n, 0), 3) for n in counts]
        n_new = sum(max(n, 0) for n in counts)
        qn, kn, vn = normal(rng, tokens, q_heads, dim), normal(rng, tokens, heads, dim), normal(rng, tokens, heads, dim)
        paths = np.full((streams, most), -1, np.int32)
        for i, t in enumerate(trees):
            if t:
                leaf = int(rng.integers(0, len(t)))
                path = [j for j in range(len(t)) if t[leaf] >> j & 1]
                paths[i, :len(path)] = path
        set_(fresh, np.array(counts, np.int32))
        set_(kept, paths)
        set_(seen, np.array([m for t in trees for m in t] + [0] * (tokens - n_new), np.uint64))
        for p, a in ((q, qn), (k, kn), (v, vn)):
            set_(p.base, np.concatenate([a.reshape(-1).view(np.uint16), np.full(8, 0x7E00, np.uint16)]))
        set_(out.base, np.full(out.n, 0x7E00, np.uint16))
        dev.check(dev.lib.mlvc_hip_graph_launch(graph, stream))
        dev.check(dev.lib.mlvc_hip_stream_synchronize(stream))
        want = plan.host(length, counts, tokens, np.array([m for t in trees for m in t] + [0] * tokens, np.uint64))
        plan.compare(want, tokens)
        assert want["lacking"] == 0
        got, at = out.get(), 0
        for i, t in enumerate(trees):
            if not t:
                continue
            n = len(t)
            kk, vv = np.concatenate([held_k[i], kn[at:at + n]]), np.concatenate([held_v[i], vn[at:at + n]])
            ref, tol = masked64(f64(qn[at:at + n]), stored64(kk, kind), stored64(vv, kind), 0.125,
                                drafts_seen(length[i] + n, t, window, sinks), tops_of(vv, kind))
            within(got[at:at + n], ref, tol, f"step {step}, stream {i}")
            path = [d for d in paths[i] if d >= 0]
            held_k[i], held_v[i] = np.concatenate([held_k[i], kn[at:at + n][path]]), np.concatenate([held_v[i], vn[at:at + n][path]])
            length[i] += len(path)
            at += n
        assert np.isnan(got[n_new:]).all()
        assert dev.get(past, (streams,), np.int32).tolist() == length
    dev.check(dev.lib.mlvc_hip_graph_destroy(graph))
    dev.check(dev.lib.mlvc_hip_stream_destroy(stream))
