"""Token operators (norm and rotation, paged cache, prompt and token
attention) against their definitions in 64 bits, through the device C ABI."""

import numpy as np
import pytest

import mlvc_hip
from devmem import Dev
from mlvc_hip import KV_E4M3, KV_F16, KV_INT8
from tokens import Cache, Padded, Prompt, Token, attend64, f64, rope64, stored64, within

pytestmark = pytest.mark.gpu

KINDS = [KV_F16, KV_E4M3, KV_INT8]


@pytest.fixture
def dev():
    d = Dev()
    yield d
    d.close()


def normal(rng, *shape):
    return rng.standard_normal(shape).astype(np.float16)


# ------------------------------------------------------------ norm and rotation

def _rope(dev, q, k, wq, wk, positions, freqs, interleaved, rot_scale=1.0, eps=1e-6, extra=0, shift=0, in_place=False):
    qp, kp = Padded(dev, q, extra, shift), Padded(dev, k, extra, shift)
    qo, ko = (qp, kp) if in_place else (Padded(dev, np.zeros_like(q), extra, shift), Padded(dev, np.zeros_like(k), extra, shift))
    d = mlvc_hip.QkNormRope(
        tokens=q.shape[0], q_heads=q.shape[1], k_heads=k.shape[1], head_dim=q.shape[2], q=qp.at, k=kp.at, q_out=qo.at,
        k_out=ko.at, q_stride=qp.stride, k_stride=kp.stride, q_out_stride=qo.stride, k_out_stride=ko.stride,
        q_weight=None if wq is None else dev.put(wq), k_weight=None if wk is None else dev.put(wk), eps=eps,
        positions=dev.put(np.asarray(positions, np.int32)), freqs=dev.put(freqs), rot_dim=2 * len(freqs),
        interleaved=int(interleaved), rot_scale=rot_scale)
    mlvc_hip.qk_norm_rope(d)
    return qo.get(), ko.get()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,q_heads,k_heads,dim,rot,norm,extra,shift", [
    (1, 16, 4, 64, 64, True, 0, 0),
    (7, 16, 4, 64, 32, True, 8, 8),
    (33, 8, 1, 128, 128, False, 0, 0),
    (2049, 3, 2, 128, 32, True, 64, 0),   # four tokens a workgroup, the last one short
    (5, 2, 2, 256, 160, True, 0, 0),
    (4, 3, 1, 96, 96, True, 0, 0),        # rows of 12 lanes
    (4, 3, 1, 96, 48, True, 0, 0),        # half layout: 24 apart
    (4, 3, 1, 96, 20, True, 0, 0),        # pairs that end inside a lane
    (9, 3, 2, 128, 64, True, 1, 3),       # off 16 bytes
    (3, 5, 2, 33, 10, True, 0, 0),
    (2, 1, 1, 512, 512, True, 0, 0),
    (3, 4, 4, 64, 0, True, 0, 0),         # norm alone
    (6, 5, 0, 128, 128, True, 0, 0),      # no keys
])
def test_norm_and_rotation(dev, rng, tokens, q_heads, k_heads, dim, rot, norm, interleaved, extra, shift):
    q, k = normal(rng, tokens, q_heads, dim) * np.float16(1.5), normal(rng, tokens, k_heads, dim)
    wq, wk = (normal(rng, dim) * np.float16(0.1) + np.float16(1) if norm else None for _ in range(2))
    positions = rng.integers(0, 70000, tokens)
    freqs, _ = mlvc_hip.rope_frequencies(rot)
    got = _rope(dev, q, k, wq, wk, positions, freqs, interleaved, extra=extra, shift=shift)
    for name, g, x, w in (("q", got[0], q, wq), ("k", got[1], k, wk)):
        want, tol = rope64(x, w, 1e-6, positions, freqs, interleaved, 1.0)
        within(g, want, tol, name)


@pytest.mark.parametrize("dim,shift", [(128, 0), (64, 0), (128, 1)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_in_place_scaled_and_far(dev, rng, dim, shift, interleaved):
    q, k = normal(rng, 11, 6, dim), normal(rng, 11, 2, dim)
    positions = np.array([0, 1, 2, 1000, 65535, 65536, 131071, 1000000, 2000000, -5, 77])
    freqs, scale = mlvc_hip.rope_frequencies(dim, 1e6, mlvc_hip.ROPE_BANDS, 4.0, 4096)
    got = _rope(dev, q, k, None, None, positions, freqs, interleaved, rot_scale=scale, shift=shift, in_place=True)
    for g, x in zip(got, (q, k)):
        want, tol = rope64(x, None, 0, positions, freqs, interleaved, scale)
        within(g, want, tol)


@pytest.mark.parametrize("tokens", [2050, 4111, 8191, 8193, 10007])
@pytest.mark.parametrize("in_place", [False, True])
def test_norm_and_rotation_of_many_tokens(dev, rng, tokens, in_place):
    """More tokens than the GPU holds workgroups: one to several of them each, some with one less."""
    q, k, w = normal(rng, tokens, 2, 64), normal(rng, tokens, 1, 64), normal(rng, 64)
    positions = rng.integers(0, 70000, tokens)
    freqs, _ = mlvc_hip.rope_frequencies(32)
    got = _rope(dev, q, k, w, w, positions, freqs, False, in_place=in_place)
    for g, x in zip(got, (q, k)):
        want, tol = rope64(x, w, 1e-6, positions, freqs, False, 1.0)
        within(g, want, tol)


def test_norm_of_zero_and_large_rows(dev):
    q = np.zeros((3, 2, 64), np.float16)
    q[1] = 60000.0
    q[2] = 6e-8
    w = np.ones(64, np.float16)
    freqs = np.zeros(0)
    got, _ = _rope(dev, q, q[:, :0], w, None, [0, 0, 0], freqs, False)
    want, tol = rope64(q, w, 1e-6, np.zeros(3), freqs, False, 1.0)
    within(got, want, tol)


# ------------------------------------------------------------ cache

def _heavy(rng, *shape):
    return (rng.standard_normal(shape) * np.exp2(rng.uniform(-12, 6, (*shape[:-1], 1)))).astype(np.float16)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,dim,page,extra,shift", [
    (8, 128, 16, 0, 0), (3, 64, 48, 16, 8), (2, 256, 32, 0, 0), (5, 96, 64, 8, 0),
    (2, 24, 16, 0, 0), (1, 512, 16, 0, 0), (3, 128, 16, 3, 1),
])
def test_cache_round_trip(dev, rng, kind, heads, dim, page, extra, shift):
    tokens, pages = 53, 9
    k, v = _heavy(rng, tokens, heads, dim), _heavy(rng, tokens, heads, dim)
    k[3], v[5, 0] = 0, 0                  # zero rows
    k[7, :, :] = np.float16(6e-8)         # the smallest subnormal throughout
    v[8, 0, ::2], v[8, 0, 1::2] = 1.0, 0.5  # INT8 ties: half the largest is 63.5 steps
    k[9, 0, 0] = np.float16(65504)
    k[10, heads - 1, 1], v[11, 0, dim - 1] = np.inf, np.nan
    slots = rng.permutation(pages * page)[:tokens]
    cache = Cache(dev, kind, pages, page, heads, dim)
    cache.write(k, v, slots, extra, shift)
    order = rng.permutation(tokens)
    for x, g in zip((k, v), cache.read(slots[order], extra, shift)):
        want = stored64(x, kind)[order]
        if kind == KV_F16:
            assert np.array_equal(g.view(np.uint16), x[order].view(np.uint16))
        else:
            with np.errstate(invalid="ignore"):
                within(g, want, np.abs(want) * (2.0 ** -11 + 2.0 ** -23) + 2.0 ** -25)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [128, 24])
def test_cache_slots_outside_are_skipped(dev, rng, kind, dim):
    cache = Cache(dev, kind, 3, 16, 2, dim)
    x = normal(rng, 4, 2, dim)
    first = np.arange(0, 48)
    cache.write(np.zeros((48, 2, dim), np.float16), np.zeros((48, 2, dim), np.float16), first)
    cache.write(x, x, [5, -1, 48, 2 ** 31 - 1])
    k, v = cache.read(np.concatenate([first, [-1, 48, 2 ** 31 - 1, -2 ** 31]]))
    want = np.zeros((52, 2, dim))
    want[5] = stored64(x, kind)[0]
    for g in (k, v):
        within(g, want, np.abs(want) * 2.0 ** -10 + 2.0 ** -25)


def test_cache_past_32_bits(dev, rng):
    """5 GB of keys: rows beyond 2^32 bytes, written, read and attended."""
    pages, page, heads, dim = 40000, 16, 64, 128
    cache = Cache.__new__(Cache)
    cache.dev, cache.kind, cache.page_size, cache.heads, cache.dim, cache.pages = dev, KV_INT8, page, heads, dim, pages
    cache.desc = mlvc_hip.KvCache(kind=KV_INT8, pages=pages, page_size=page, heads=heads, head_dim=dim)
    nbytes, scales = mlvc_hip.kv_cache_bytes(cache.desc)
    assert nbytes > 2 ** 32
    cache.desc.k, cache.desc.v = dev.alloc(nbytes), dev.alloc(nbytes)
    cache.desc.k_scale, cache.desc.v_scale = dev.alloc(scales), dev.alloc(scales)
    table = np.array([[39999, 0, 33333, 17]])
    slots = np.concatenate([p * page + np.arange(page) for p in table[0]])
    k, v, q = normal(rng, 64, heads, dim), normal(rng, 64, heads, dim), normal(rng, 1, heads, dim)
    cache.write(k, v, slots)
    gk, gv = cache.read(slots)
    within(gk, stored64(k, KV_INT8), 2.0 ** -10 * np.abs(f64(k)).max())
    want, tol = attend64(f64(q), stored64(k, KV_INT8)[:57], stored64(v, KV_INT8)[:57], 0.09, False)
    within(Token(cache, q, table, [57], 0.09).run(), want, tol)


# ------------------------------------------------------------ prompt attention

def _prompt(dev, rng, queries, keys, q_heads, kv_heads, dim, causal, extra=0, shift=0, spread=1.0):
    q = normal(rng, sum(queries), q_heads, dim) * np.float16(spread)
    k, v = (normal(rng, sum(keys), kv_heads, dim) for _ in range(2))
    got = Prompt(dev, q, k, v, queries, keys, causal, dim ** -0.5, extra, shift).run()
    i = j = 0
    for nq, nk in zip(queries, keys):
        want, tol = attend64(f64(q[i:i + nq]), f64(k[j:j + nk]), f64(v[j:j + nk]), dim ** -0.5, causal)
        within(got[i:i + nq], want, tol, f"sequence of {nq} on {nk}")
        i, j = i + nq, j + nk


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("queries,keys", [
    ([1], [1]), ([2], [2]), ([31], [31]), ([33], [33]), ([128], [128]), ([129], [129]), ([257], [257]),
    ([1, 240, 0, 65, 3], [1, 240, 7, 65, 3]),
    ([1, 17, 130], [300, 64, 131]),      # behind what came before
    ([40, 200, 5], [7, 64, 0]),          # more queries than keys: rows that see nothing
])
def test_prompt_lengths(dev, rng, queries, keys, dim, causal):
    _prompt(dev, rng, queries, keys, 2, 1, dim, causal)


@pytest.mark.parametrize("dim,q_heads,kv_heads,extra,shift", [
    (64, 4, 4, 0, 0), (128, 8, 1, 0, 0), (64, 6, 2, 64, 0), (128, 5, 5, 8, 16), (128, 16, 1, 0, 0),
    (64, 3, 1, 1, 0), (128, 2, 2, 0, 1),                       # off 16 bytes
    (32, 4, 2, 0, 0), (96, 3, 3, 0, 0), (40, 2, 1, 3, 1), (256, 2, 1, 0, 0), (1, 2, 1, 0, 0), (512, 1, 1, 0, 0),
])
@pytest.mark.parametrize("causal", [False, True])
def test_prompt_heads_and_strides(dev, rng, dim, q_heads, kv_heads, extra, shift, causal):
    _prompt(dev, rng, [70, 19], [70, 33], q_heads, kv_heads, dim, causal, extra, shift)


@pytest.mark.parametrize("dim", [64, 128, 96])
def test_prompt_peaked_and_flat(dev, rng, dim):
    """Scores from one dominant key (hundreds apart) to all equal."""
    _prompt(dev, rng, [150], [150], 2, 2, dim, True, spread=60.0)
    _prompt(dev, rng, [150], [150], 2, 2, dim, True, spread=0.0)


@pytest.mark.parametrize("dim", [64, 128, 96])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_prompt_unseen_rows_do_not_reach(dev, rng, dim, bad):
    """Non-finite keys and values past a query's place, and in a neighbouring sequence."""
    queries, keys = [100, 90], [100, 90]
    q, k, v = (normal(rng, 190, 2, dim) for _ in range(3))
    k[60], v[61, 0, 3], v[99, 1, dim - 1] = bad, bad, bad
    k[100:], v[100:] = bad, bad
    got = Prompt(dev, q, k, v, queries, keys, True, dim ** -0.5).run()
    want, tol = attend64(f64(q[:60]), f64(k[:60]), f64(v[:60]), dim ** -0.5, True)
    within(got[:60], want, tol)
    # Value columns without the non-finite element stay finite where the keys are.
    k[60] = 0
    got = Prompt(dev, q, k, v, queries, keys, True, dim ** -0.5).run()[:100]
    clean = v[:100].copy()
    clean[61, 0, 3], clean[99, 1, dim - 1] = 0, 0
    want, tol = attend64(f64(q[:100]), f64(k[:100]), f64(clean), dim ** -0.5, True)
    want[61:, 0, 3], want[99:, 1, dim - 1] = bad, bad
    assert np.array_equal(np.isnan(got), np.isnan(want)) or not np.isnan(bad)
    assert not np.isfinite(got[61:, 0, 3]).any() and not np.isfinite(got[99:, 1, dim - 1]).any()
    keep = np.isfinite(want)
    assert np.isfinite(got[keep]).all()
    within(np.where(keep, got, 0), np.where(keep, want, 0), tol)


@pytest.mark.parametrize("dim", [64, 128, 32])
def test_prompt_cut_starts(dev, rng, dim):
    """longest_q and starts beyond the tensors are cut; rows outside stay as they were."""
    q, k, v = normal(rng, 50, 2, dim), normal(rng, 40, 2, dim), normal(rng, 40, 2, dim)
    starts = ([3, 23, 60], [5, 30, 90])
    got = Prompt(dev, q, k, v, [20, 27], [25, 10], True, 0.1, longest=24, starts=starts).run()
    assert np.isnan(got[:3]).all() and np.isnan(got[23 + 24:]).all()
    want, tol = attend64(f64(q[3:23]), f64(k[5:30]), f64(v[5:30]), 0.1, True)
    within(got[3:23], want, tol)
    want, tol = attend64(f64(q[23:50]), f64(k[30:40]), f64(v[30:40]), 0.1, True)
    within(got[23:47], want[:24], tol[:24])


def test_prompt_strides_past_32_bits(dev, rng):
    """Rows 2^25 halves apart: offsets beyond 2^32 bytes."""
    dim, n, stride = 64, 80, 1 << 25
    k, v, q = (normal(rng, n, 1, dim) for _ in range(3))
    base = dev.alloc(2 * stride * n)
    for i in range(n):
        row = np.concatenate([k[i], v[i], q[i]]).astype(np.float16)
        dev.check(dev.lib.mlvc_hip_memcpy_h2d(base.value + 2 * stride * i, row.ctypes.data, row.nbytes, None))
        dev.check(dev.lib.mlvc_hip_stream_synchronize(None))
    p = Prompt(dev, q, k, v, [n], [n], True, 0.125)
    p.desc.k, p.desc.v, p.desc.q = base.value, base.value + 2 * dim, base.value + 4 * dim
    p.desc.q_stride = p.desc.k_stride = p.desc.v_stride = stride
    want, tol = attend64(f64(q), f64(k), f64(v), 0.125, True)
    within(p.run(), want, tol)


# ------------------------------------------------------------ token attention

def _streams(dev, rng, kind, lengths, heads, dim, page, spare=2):
    """A cache with the streams' contexts in shuffled pages, its table, and what it stands for."""
    used = [-(-n // page) for n in lengths]
    pages = sum(used) + spare
    cache = Cache(dev, kind, pages, page, heads, dim)
    free = list(rng.permutation(pages))
    table = np.full((len(lengths), max(max(used), 1)), -1)
    ks, vs = [], []
    for i, n in enumerate(lengths):
        table[i, :used[i]] = [free.pop() for _ in range(used[i])]
        j = np.arange(n)
        k, v = normal(rng, n, heads, dim), normal(rng, n, heads, dim) * np.float16(3)
        if n:
            cache.write(k, v, table[i, j // page] * page + j % page)
        ks.append(stored64(k, kind) if n else np.zeros((0, heads, dim)))
        vs.append(stored64(v, kind) if n else np.zeros((0, heads, dim)))
    return cache, table, ks, vs


def _check_tokens(got, q, ks, vs, lengths, scale):
    for i, n in enumerate(lengths):
        want, tol = attend64(f64(q[i:i + 1]), ks[i][:n], vs[i][:n], scale, False)
        within(got[i:i + 1], want, tol, f"stream {i} of {n}")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("q_heads,heads,dim,page,lengths", [
    (4, 1, 64, 16, [0, 1, 15, 16, 17, 31, 33, 64, 100]),
    (4, 4, 128, 48, [1, 47, 48, 49, 95, 97, 300]),
    (8, 1, 128, 16, [515, 3, 0, 1025]),
    (16, 1, 64, 64, [700]), (20, 1, 128, 32, [130, 9]), (34, 2, 64, 16, [257]),
    (6, 3, 128, 16, [2500, 1]),
    (3, 3, 32, 16, [50, 0]), (2, 1, 96, 16, [300]), (2, 2, 256, 32, [70]), (1, 1, 512, 16, [65]), (5, 1, 8, 16, [33]),
])
def test_tokens(dev, rng, kind, q_heads, heads, dim, page, lengths):
    cache, table, ks, vs = _streams(dev, rng, kind, lengths, heads, dim, page)
    q = normal(rng, len(lengths), q_heads, dim)
    _check_tokens(Token(cache, q, table, lengths, dim ** -0.5).run(), q, ks, vs, lengths, dim ** -0.5)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("extra,shift", [(8, 0), (0, 1), (5, 3)])
def test_tokens_strides(dev, rng, kind, extra, shift):
    lengths = [90, 33]
    cache, table, ks, vs = _streams(dev, rng, kind, lengths, 2, 128, 16)
    q = normal(rng, 2, 8, 128)
    _check_tokens(Token(cache, q, table, lengths, 0.1, extra=extra, shift=shift).run(), q, ks, vs, lengths, 0.1)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 96])
def test_tokens_scores_far_apart(dev, rng, kind, dim):
    """Rows of very different magnitude: scores hundreds apart, value scales 2^18 apart."""
    n = 400
    cache = Cache(dev, kind, 30, 16, 1, dim)
    k, v, q = _heavy(rng, n, 1, dim), _heavy(rng, n, 1, dim), normal(rng, 1, 4, dim) * np.float16(4)
    table = rng.permutation(30)[None, :25]
    j = np.arange(n)
    cache.write(k, v, table[0, j // 16] * 16 + j % 16)
    for scale in (dim ** -0.5, 0.01, -0.05):
        got = Token(cache, q, table, [n], scale).run()
        _check_tokens(got, q, [stored64(k, kind)], [stored64(v, kind)], [n], scale)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 96])
def test_tokens_unseen_places_do_not_reach(dev, rng, kind, dim):
    """What the pages hold past a length, lengths past the bounds, and pages outside the cache."""
    lengths = [40, 37]
    cache, table, ks, vs = _streams(dev, rng, kind, lengths, 2, dim, 16)  # unwritten places hold NaN bits and NaN scales
    q = normal(rng, 2, 4, dim)
    _check_tokens(Token(cache, q, table, lengths, 0.1).run(), q, ks, vs, lengths, 0.1)
    # Lengths are cut to `longest`, then to the table; negative is empty.
    _check_tokens(Token(cache, q, table, [1000, -3], 0.1, longest=35).run(), q, ks, vs, [35, 0], 0.1)
    _check_tokens(Token(cache, q, table[:, :2], [40, 20], 0.1, longest=10 ** 6).run(), q, ks, vs, [32, 20], 0.1)
    # A page outside the cache is not seen.
    holes = table.copy()
    holes[0, 1], holes[1, 0], holes[1, 1] = -1, cache.pages, 2 ** 31 - 1
    got = Token(cache, q, holes, lengths, 0.1).run()
    seen = [np.r_[0:16, 32:40], np.r_[32:37]]
    for i in range(2):
        want, tol = attend64(f64(q[i:i + 1]), ks[i][seen[i]], vs[i][seen[i]], 0.1, False)
        within(got[i:i + 1], want, tol)


@pytest.mark.parametrize("kind", [KV_E4M3, KV_INT8])
def test_tokens_nan_rows_show(dev, rng, kind):
    """A seen row that holds an infinity is NaN to every query, in its own head only."""
    cache = Cache(dev, kind, 2, 16, 2, 64)
    k, v = normal(rng, 20, 2, 64), normal(rng, 20, 2, 64)
    v[5, 0, 7] = np.inf
    cache.write(k, v, np.arange(20))
    got = Token(cache, normal(rng, 1, 4, 64), [[0, 1]], [20], 0.1).run()
    assert np.isnan(got[0, :2]).all() and np.isfinite(got[0, 2:]).all()


@pytest.mark.parametrize("kind", KINDS)
def test_tokens_are_repeatable(dev, rng, kind):
    """Parts are joined in a fixed order: the same bits on every call."""
    lengths = [5000, 700, 1, 2999]
    cache, table, _, _ = _streams(dev, rng, kind, lengths, 2, 64, 32)
    t = Token(cache, normal(rng, 4, 8, 64), table, lengths, 0.125)
    first = t.run().view(np.uint16)
    for _ in range(3):
        assert np.array_equal(first, t.run().view(np.uint16))


def test_token_step_captured(dev, rng):
    """Write, attend: captured once, replayed while lengths and rows change, against eager runs."""
    import ctypes as C

    lib = dev.lib
    stream, graph = C.c_void_p(), C.c_void_p()
    dev.check(lib.mlvc_hip_stream_create(C.byref(stream)))
    heads, dim, page = 2, 128, 16
    cache, table, ks, vs = _streams(dev, rng, KV_INT8, [600, 37], heads, dim, page, spare=4)
    table = np.concatenate([table, [[-1], [-1]]], 1)
    table[0, -1], table[1, 3] = sorted(set(range(cache.pages)) - set(table.ravel()))[:2]
    q = normal(rng, 2, 8, dim)
    t = Token(cache, q, table, [600, 37], 0.1, longest=608)
    k, v = Padded(dev, np.zeros((2, heads, dim), np.float16)), Padded(dev, np.zeros((2, heads, dim), np.float16))
    rows = cache.rows(k, v, [-1, -1])
    dev.check(lib.mlvc_hip_capture_begin(stream))
    mlvc_hip.kv_write(cache.desc, rows, stream)
    mlvc_hip.attention_token(t.desc, stream)
    dev.check(lib.mlvc_hip_capture_end(stream, C.byref(graph)))
    lengths = [600, 37]
    try:
        for step in range(4):
            new_k, new_v = normal(rng, 2, heads, dim), normal(rng, 2, heads, dim)
            slots = np.array([table[i, n // page] * page + n % page for i, n in enumerate(lengths)], np.int32)
            lengths = [n + 1 for n in lengths]
            for at, a in ((k.at, new_k), (v.at, new_v), (rows.slots, slots), (t.lengths, np.array(lengths, np.int32))):
                dev.check(lib.mlvc_hip_memcpy_h2d(at, a.ctypes.data, a.nbytes, stream))
                dev.check(lib.mlvc_hip_stream_synchronize(stream))
            dev.check(lib.mlvc_hip_graph_launch(graph, stream))
            dev.check(lib.mlvc_hip_stream_synchronize(stream))
            got = t.out.get()
            for i in range(2):
                ks[i] = np.concatenate([ks[i], stored64(new_k[i:i + 1], KV_INT8)])
                vs[i] = np.concatenate([vs[i], stored64(new_v[i:i + 1], KV_INT8)])
            _check_tokens(got, q, ks, vs, lengths, 0.1)
            assert np.array_equal(got.view(np.uint16), Token(cache, q, table, lengths, 0.1, longest=608).run().view(np.uint16))
    finally:
        dev.check(lib.mlvc_hip_graph_destroy(graph))
        dev.check(lib.mlvc_hip_stream_destroy(stream))


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("queries,keys,q_heads", [
    ([130], [130], 64), ([97, 1, 64], [210, 7, 64], 64),       # a few queries a workgroup, keys in four groups
    ([261], [261], 64), ([200, 77], [333, 50], 64),            # 128 queries, keys in groups
    ([530], [700], 64), ([1100, 3], [1100, 65], 64),           # 128 queries, one group and several
    ([4100], [4100], 32), ([4100], [4300], 32),                # 256 queries
])
def test_prompt_tiles(dev, rng, queries, keys, q_heads, dim, causal):
    """Sizes for every tile shape: a sample of the queries, with the first and last of each sequence."""
    q = normal(rng, sum(queries), q_heads, dim)
    k, v = (normal(rng, sum(keys), 2, dim) for _ in range(2))
    got = Prompt(dev, q, k, v, queries, keys, causal, dim ** -0.5).run()
    assert np.isfinite(got).all()
    i = j = 0
    for nq, nk in zip(queries, keys):
        rows = np.unique(np.r_[0, nq - 1, rng.integers(0, nq, 8)])
        heads = rng.permutation(q_heads)[:4]
        for r in rows:
            n = min(nk, max(0, nk - nq + r + 1)) if causal else nk
            for h in heads:
                g = h // (q_heads // 2)
                want, tol = attend64(f64(q[i + r:i + r + 1, h:h + 1]), f64(k[j:j + n, g:g + 1]), f64(v[j:j + n, g:g + 1]),
                                     dim ** -0.5, False)
                within(got[i + r:i + r + 1, h:h + 1], want, tol, f"query {r} of {nq} on {nk}, head {h}")
        i, j = i + nq, j + nk


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,q_heads", [(130, 64), (261, 64), (530, 64), (1100, 64)])
def test_prompt_tiles_unseen_rows(dev, rng, n, q_heads, dim):
    """A value that is not finite reaches the queries from its place on, in every tile shape."""
    q, k, v = normal(rng, n, q_heads, dim), normal(rng, n, 1, dim), normal(rng, n, 1, dim)
    bad = {n - 2: np.nan, n // 2: np.inf, n // 2 + 1: -np.inf}
    for at, x in bad.items():
        v[at, 0, at % dim] = x
    got = Prompt(dev, q, k, v, [n], [n], True, dim ** -0.5).run()
    for column in {at % dim for at in bad}:
        at = min(a for a in bad if a % dim == column)  # two of them may share a column
        assert np.isfinite(got[:at, :, column]).all() and not np.isfinite(got[at:, :, column]).any()
    columns = np.setdiff1d(np.arange(dim), [at % dim for at in bad])
    assert np.isfinite(got[:, :, columns]).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("sequences,q_heads,kv_heads,longest", [
    (23, 32, 4, None),     # a CU holds several workgroups, an XCD whole heads
    (55, 10, 5, None),     # heads that the XCDs do not divide
    (64, 16, 16, 5000),    # a bound on the queries far above them
    (90, 8, 2, None),      # more sequences than a wave has lanes
])
def test_prompt_many_ragged_sequences(dev, rng, dim, causal, sequences, q_heads, kv_heads, longest):
    """Sequences of 0 to 300 queries on fewer or more keys: every query is answered once, by its own keys."""
    queries = [int(n) for n in rng.choice([0, 1, 5, 31, 128, 129, 300], sequences)]
    keys = [max(0, n + int(more)) for n, more in zip(queries, rng.choice([0, 0, -40, 3, 64, 500], sequences))]
    q = normal(rng, sum(queries), q_heads, dim)
    k, v = normal(rng, sum(keys), kv_heads, dim), normal(rng, sum(keys), kv_heads, dim)
    got = Prompt(dev, q, k, v, queries, keys, causal, dim ** -0.5, longest=longest).run()
    assert np.isfinite(got).all()
    sq, sk = np.cumsum([0] + queries), np.cumsum([0] + keys)
    for head in {0, q_heads // 2 + 1}:
        kv = head // (q_heads // kv_heads)
        for n in range(sequences):
            a, b = slice(sq[n], sq[n + 1]), slice(sk[n], sk[n + 1])
            want, tol = attend64(f64(q[a, head:head + 1]), f64(k[b, kv:kv + 1]), f64(v[b, kv:kv + 1]), dim ** -0.5, causal)
            within(got[a, head:head + 1], want, tol)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lengths", [[130] * 70, [5] * 129 + [700], [900] + [0, 1, 40] * 43])
def test_prompt_more_sequences_than_lanes(dev, rng, dim, lengths):
    """Alike ones, and a long one behind or before many short ones, over more than one and two waves' lanes."""
    q, k, v = (normal(rng, sum(lengths), heads, dim) for heads in (10, 2, 2))
    got = Prompt(dev, q, k, v, lengths, lengths, True, dim ** -0.5).run()
    assert np.isfinite(got).all()
    ends = np.cumsum([0] + lengths)
    for n in range(len(lengths)):
        at = slice(ends[n], ends[n + 1])
        want, tol = attend64(f64(q[at, 7:8]), f64(k[at, 1:]), f64(v[at, 1:]), dim ** -0.5, True)
        within(got[at, 7:8], want, tol)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("queries,keys,q_heads", [
    ([700, 500], [1100, 500], 16),          # tiles that just fit the CUs
    ([95, 0, 97, 960], [95, 300, 96, 960], 16),
    ([450, 449, 1], [900, 3, 70], 24),
])
def test_prompt_tiles_that_fit_the_gpu(dev, rng, dim, causal, queries, keys, q_heads):
    q = normal(rng, sum(queries), q_heads, dim)
    k, v = normal(rng, sum(keys), 8, dim), normal(rng, sum(keys), 8, dim)
    v[sum(keys) - 2, :, 5] = np.inf
    got = Prompt(dev, q, k, v, queries, keys, causal, dim ** -0.5).run()
    sq, sk = np.cumsum([0] + queries), np.cumsum([0] + keys)
    columns = np.delete(np.arange(dim), 5)
    assert np.isfinite(got[:, :, columns]).all()
    for head in (0, q_heads - 1):
        kv = head // (q_heads // 8)
        for n in range(len(queries)):
            a, b = slice(sq[n], sq[n + 1]), slice(sk[n], sk[n + 1])
            want, tol = attend64(f64(q[a, head:head + 1]), f64(k[b, kv:kv + 1]), f64(v[b, kv:kv + 1]), dim ** -0.5, causal)
            within(got[a, head:head + 1][:, :, columns], want[:, :, columns], tol[:, :, columns])
            assert np.array_equal(np.isfinite(got[a, head, 5]), np.isfinite(want[:, 0, 5]))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,dim,lengths", [
    (2, 64, [0, 30000, 1, 700]),          # one stream in many shares, others inside one
    (1, 128, [40] * 100 + [2000]),        # more streams than a wave has lanes, many in a share
    (4, 64, [2048, 4096, 8192, 0, 5]),    # shares that end where streams do
])
def test_tokens_shares(dev, rng, kind, heads, dim, lengths):
    cache, table, ks, vs = _streams(dev, rng, kind, lengths, heads, dim, 64)
    q = normal(rng, len(lengths), 2 * heads, dim)
    _check_tokens(Token(cache, q, table, lengths, dim ** -0.5).run(), q, ks, vs, lengths, dim ** -0.5)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,dim,streams,longest", [
    (4, 128, 48, 2048),     # half as many contexts as CUs and more
    (8, 64, 100, 4096),     # three times as many
    (3, 96, 70, 2047),      # heads without matrix cores
])
def test_tokens_whole_contexts_of_large_batches(dev, rng, kind, heads, dim, streams, longest):
    """Contexts past 1024 tokens that are not cut, beside short and empty ones; a smaller batch fits the same workspace."""
    lengths = [int(n) for n in rng.choice([0, 1, 33, 250], streams)]
    lengths[3], lengths[streams - 1] = longest, longest - 40
    cache, table, ks, vs = _streams(dev, rng, kind, lengths, heads, dim, 32)
    q = normal(rng, streams, heads, dim)
    call = Token(cache, q, table, lengths, dim ** -0.5)
    _check_tokens(call.run(), q, ks, vs, lengths, dim ** -0.5)
    call.desc.streams = 5
    assert mlvc_hip.attention_token_workspace_bytes(call.desc) <= call.desc.workspace_bytes
    _check_tokens(call.run()[:5], q[:5], ks[:5], vs[:5], lengths[:5], dim ** -0.5)
