"""Attention over latent tokens at the ends of its numbers' range: values of
zero, weights far below the largest, infinities."""

import numpy as np
import pytest

from devmem import Dev
from mlvc_hip import KV_E4M3, KV_F16, KV_INT8
from tokens import Cache, Prompt, Token, attend64, f64, stored64, within

pytestmark = pytest.mark.gpu

KINDS = [KV_F16, KV_E4M3, KV_INT8]


@pytest.fixture
def dev():
    d = Dev()
    yield d
    d.close()


def normal(rng, *shape):
    return rng.standard_normal(shape).astype(np.float16)


def _context(dev, rng, kind, k, v, page=32):
    """One stream's context in shuffled pages, and its table."""
    n, heads, dim = k.shape
    pages = -(-n // page)
    cache = Cache(dev, kind, pages, page, heads, dim)
    table = rng.permutation(pages)[None]
    j = np.arange(n)
    cache.write(k, v, table[0, j // page] * page + j % page)
    return cache, table


# ------------------------------------------------------------ values of zero

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 96])
@pytest.mark.parametrize("n", [1, 40, 920, 5000])
def test_tokens_of_zero_values_and_low_scores(dev, rng, kind, dim, n):
    """Every value zero and every score below -100: zeros, in a whole context and in one that is cut."""
    k = normal(rng, n, 2, dim) * np.float16(0.1) - np.float16(4)
    q = normal(rng, 1, 4, dim) * np.float16(0.1) + np.float16(4)
    cache, table = _context(dev, rng, kind, k, np.zeros_like(k))
    assert (f64(q[0]) @ f64(k[:, 0]).T).max() * dim ** -0.5 < -100
    assert np.array_equal(Token(cache, q, table, [n], dim ** -0.5).run(), np.zeros((1, 4, dim)))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 96])
def test_tokens_beside_a_stretch_of_zero_values(dev, rng, kind, dim):
    """Whole shares of a cut context with values of zero and scores below -100, beside ordinary ones."""
    n, blank = 8160, slice(2000, 4500)
    k, v = normal(rng, n, 1, dim), normal(rng, n, 1, dim)
    q = normal(rng, 1, 4, dim) * np.float16(0.1) + np.float16(4)
    k[blank] = normal(rng, 2500, 1, dim) * np.float16(0.1) - np.float16(4)
    v[blank] = 0
    cache, table = _context(dev, rng, kind, k, v)
    want, tol = attend64(f64(q), stored64(k, kind), stored64(v, kind), dim ** -0.5, False)
    within(Token(cache, q, table, [n], dim ** -0.5).run(), want, tol)


# ------------------------------------------------------------ small weights

# The matrix kernels give weights to the matrix cores in FP16, the largest as at
# least 2^12: below 2^-14, a quantum of 2^-24. So a weight is off by half of
# that, 2^-37 of the largest, beside its rounding of 2^-11 (2^-22 with a
# remainder).
LEAST = 2.0 ** -37


def _beside_a_sink(n, heads, dim):
    """Query, keys and values: key 0 has the score 0 and a value in column 0 only, all others a score 17.7
    lower (2^-25.5 of its weight) and values from 0.5 to 1.5."""
    q = np.ones((1, 1, dim), np.float16)
    k = np.full((n, heads, dim), -17.7 / 8 / dim ** 0.5, np.float16)
    v = np.random.default_rng(9).uniform(0.5, 1.5, (n, heads, dim)).astype(np.float16)
    k[0], v[0], v[0, :, 0] = 0, 0, 1
    return q, k, v


def _weighed(k, q, v, scale, rounding, least):
    """(result, tolerance) of one query [dim] on keys and values [n, dim] for weights off by `rounding` of
    themselves and by least[j] of the largest weight."""
    s = k @ q * scale
    p = np.exp(s - s.max())
    w, out = p / p.sum(), p @ v / p.sum()
    # Scores: FP32 products and sums of dim terms, the exponent's rounding; FP32 sums of n terms.
    ds = (np.abs(k) @ np.abs(q)) * abs(scale) * (len(q) + 4) * 2.0 ** -24 + np.abs(s) * 2.0 ** -22 + 2.0 ** -21
    off = w * (rounding + 2 * ds) + least / p.sum()
    tol = np.abs(out) * 2.0 ** -11 + 2.0 ** -25 + off @ (np.abs(v) + np.abs(out)) + (len(p) + 8) * 2.0 ** -24 * (w @ np.abs(v))
    return out, tol


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n", [900, 8160, 65280])
def test_tokens_of_small_weights(dev, rng, kind, dim, n):
    """Thousands of tokens that matter together and not each, beside one that dominates the sum of weights."""
    q, k, v = _beside_a_sink(n, 1, dim)
    cache, table = _context(dev, rng, kind, k, v)
    k, v = stored64(k, kind)[:, 0], stored64(v, kind)[:, 0]
    scale = dim ** -0.5 * 8
    # With a quantised cache a weight is scaled by its value's scale, and the largest of those counts.
    units = np.ones(n) if kind == KV_F16 else np.abs(v).max(-1) / (448 if kind == KV_E4M3 else 127)
    p = np.exp(k @ f64(q[0, 0]) * scale)
    # Exponents, with the scale's logarithm, are up to 2^6 in FP32: two roundings of 2^-19, times ln 2.
    want, tol = _weighed(k, f64(q[0, 0]), v, scale, 2.0 ** -22 + 2.0 ** -18, LEAST * (p * units).max() / units / p.max())
    within(Token(cache, q, table, [n], scale).run()[0, 0], want, tol)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("queries,keys,q_heads", [
    ([4], [3001], 4), ([4], [400], 4), ([130], [1300], 64), ([261], [1261], 64), ([200, 77], [933, 1050], 64),
    ([530], [1700], 64), ([1100, 3], [1100, 2065], 64), ([4100], [4100], 32),
])
def test_prompt_of_small_weights(dev, rng, queries, keys, q_heads, dim, causal):
    """The same in every tile shape, the dominating key first in each sequence."""
    parts = [_beside_a_sink(n, 2, dim) for n in keys]
    k, v = (np.concatenate([p[i] for p in parts]) for i in (1, 2))
    q = np.ones((sum(queries), q_heads, dim), np.float16)
    scale = dim ** -0.5 * 8
    got = Prompt(dev, q, k, v, queries, keys, causal, scale).run()
    i = j = 0
    for nq, nk in zip(queries, keys):
        for r in np.unique(np.r_[0, nq // 2, nq - 1]):
            n = nk - nq + r + 1 if causal else nk
            for head in (0, q_heads - 1):
                at = slice(j, j + n), head // (q_heads // 2)
                want, tol = _weighed(f64(k[at]), f64(q[0, 0]), f64(v[at]), scale, 2.0 ** -11, LEAST)
                within(got[i + r, head], want, tol, f"query {r} of {nq} on {nk}, head {head}")
        i, j = i + nq, j + nk


# ------------------------------------------------------------ large scores

def _far_apart(rng, n, heads, dim):
    """Keys of one value throughout, different ones 16 apart at least; two largest ones, alike."""
    size = rng.permutation(n).astype(np.float16) * np.float16(24)
    order = np.argsort(size)
    size[order[-2]] = size[order[-1]]
    k = np.repeat(size, heads * dim).reshape(n, heads, dim)
    return k, normal(rng, n, heads, dim), size


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 96])
@pytest.mark.parametrize("size", [0.5, 4.0, 60.0, 60000.0, -60000.0])
@pytest.mark.parametrize("n", [900, 2600])
def test_tokens_of_large_scores(dev, rng, kind, dim, size, n):
    k, v, sizes = _far_apart(rng, n, 1, dim)
    cache, table = _context(dev, rng, kind, k, v)
    q = np.full((1, 4, dim), size, np.float16)
    seen = sizes * np.sign(size)
    at = np.flatnonzero(seen == seen.max())
    v = stored64(v, kind)[at, 0]
    want = v.mean(0)
    got = Token(cache, q, table, [n], 1.0).run()
    # Beside the result's rounding, a weight through the logarithm of its value's scale: an exponent of up to
    # 2^6 in FP32, off by 2^-18 from the logarithm and 2^-19 from either of two sums.
    for head in range(4):
        within(got[0, head], want, np.abs(want) * 2.0 ** -11 + np.abs(v).mean(0) * 2.0 ** -17 + 2.0 ** -25)


@pytest.mark.parametrize("dim", [64, 128, 96])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("size", [0.5, 4.0, 60.0, 60000.0, -60000.0])
@pytest.mark.parametrize("queries,keys,q_heads", [([3], [900], 4), ([530], [1700], 64), ([1100], [1100], 64)])
def test_prompt_of_large_scores(dev, rng, queries, keys, q_heads, dim, causal, size):
    """Scores up to 2^36, further apart than FP32's rounding of them: the largest key's value, or the mean of two."""
    n, nq = keys[0], queries[0]
    k, v, sizes = _far_apart(rng, n, 2, dim)
    q = np.full((nq, q_heads, dim), size, np.float16)
    got = Prompt(dev, q, k, v, queries, keys, causal, 1.0).run()
    for r in np.unique(np.r_[0, nq // 2, nq - 1, rng.integers(0, nq, 5)]):
        seen = sizes[:n - nq + r + 1 if causal else n] * np.sign(size)
        at = np.flatnonzero(seen == seen.max())
        for head in (0, q_heads - 1):
            # Alike weights, rounded to FP16 alike, over a sum that is not; then the result's rounding.
            want = f64(v[at, head // (q_heads // 2)]).mean(0)
            within(got[r, head], want, np.abs(want) * (2.0 ** -10 + 2.0 ** -20) + 2.0 ** -25, f"query {r}, head {head}")



# ------------------------------------------------------------ infinities

def _with_odd_values(rng, n, heads, dim, peaked):
    """Keys, values with infinities and NaN, the values without them, and what each column of head 0 holds:
    {column: [(place, value), ...]}. One odd value's key has a score far below all others; peaked: the last
    key's lies far above, so that every other weight is 0 in FP32."""
    k, v = normal(rng, n, heads, dim), normal(rng, n, heads, dim)
    k[n // 2] = -60
    if peaked:
        k[n - 1] = 60
    odd = {5: [(3, np.inf)], 9: [(n - 1, -np.inf)], 20: [(n // 3, np.nan)], 30: [(6, np.inf), (n - 2, -np.inf)],
           40: [(n // 2, -np.inf)], dim - 1: [(n // 2, np.inf), (0, np.inf)]}
    clean = v.copy()
    for column, places in odd.items():
        for at, x in places:
            v[at, 0, column], clean[at, 0, column] = x, 0
    return k, v, clean, odd


def _sum_of(seen):
    """A weighted sum of such values: however small a weight, it is not 0."""
    return np.float64(0) + sum(np.float64(x) for x in seen)


@pytest.mark.parametrize("dim", [64, 128, 96])
@pytest.mark.parametrize("n", [40, 900, 5000])
@pytest.mark.parametrize("peaked", [False, True])
@pytest.mark.parametrize("extra,shift", [(0, 0), (0, 1)])
def test_tokens_of_infinite_values(dev, rng, dim, n, peaked, extra, shift):
    """An FP16 cache: a seen infinity is the result, opposite ones and NaN are NaN, in their columns and head only."""
    k, v, clean, odd = _with_odd_values(rng, n, 2, dim, peaked)
    q = normal(rng, 1, 4, dim) * np.float16(0.1) + np.float16(4)
    cache, table = _context(dev, rng, KV_F16, k, v)
    got = Token(cache, q, table, [n], dim ** -0.5, extra=extra, shift=shift).run()
    want, tol = attend64(f64(q), f64(k), f64(clean), dim ** -0.5, False)
    with np.errstate(invalid="ignore"):
        for column, places in odd.items():
            want[0, :2, column] = _sum_of(x for _, x in places)
    with np.errstate(invalid="ignore"):
        within(got, want, tol)
    same = np.isinf(want)
    assert np.array_equal(np.isnan(want), np.isnan(got)) and np.array_equal(got[same], want[same])


@pytest.mark.parametrize("dim", [64, 128, 96])
@pytest.mark.parametrize("n", [40, 5000])
def test_tokens_of_infinite_keys(dev, rng, dim, n):
    """An FP16 cache: a key with an infinity scores +inf (NaN) or -inf (not there), by the sign of the query's value."""
    k, v, q = normal(rng, n, 1, dim), normal(rng, n, 1, dim), normal(rng, 1, 4, dim)
    k[7, 0, 3] = np.inf
    q[0, :, 3] = [1, -1, 2, -2]
    cache, table = _context(dev, rng, KV_F16, k, v)
    got = Token(cache, q, table, [n], dim ** -0.5).run()
    rest = np.arange(n) != 7
    want, tol = attend64(f64(q), f64(k[rest]), f64(v[rest]), dim ** -0.5, False)
    want[0, ::2] = np.nan
    with np.errstate(invalid="ignore"):
        within(got, want, tol)
    assert np.isnan(got[0, ::2]).all()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [64, 128, 96])
@pytest.mark.parametrize("peaked", [False, True])
@pytest.mark.parametrize("queries,keys,q_heads", [
    ([3], [3001], 4), ([4], [400], 4), ([130], [1300], 64), ([261], [261], 64), ([200, 77], [933, 1050], 64),
    ([530], [530], 64), ([1100, 65], [1100, 2065], 64), ([4100], [4100], 32),
])
def test_prompt_of_infinite_values(dev, rng, queries, keys, q_heads, dim, causal, peaked):
    """A seen infinity is the result, opposite ones and NaN are NaN, in their columns, sequence and key head
    only and from their place on, in every tile shape and whatever the tile."""
    parts = [_with_odd_values(rng, n, 2, dim, False) for n in keys]
    for n, part in zip(keys, parts):
        if peaked:
            part[0][n // 4] = 60
    k, v, clean = (np.concatenate([p[i] for p in parts]) for i in range(3))
    q = normal(rng, sum(queries), q_heads, dim) * np.float16(0.1) + np.float16(4)
    got = Prompt(dev, q, k, v, queries, keys, causal, dim ** -0.5).run()
    i = j = 0
    for nq, nk, part in zip(queries, keys, parts):
        places = sorted({at for column in part[3].values() for at, _ in column} | {nk // 4})
        rows = [r + nq - nk for at in places for r in (at - 1, at)] + [0, nq - 1] + rng.integers(0, nq, 4).tolist()
        for r in sorted({r for r in rows if 0 <= r < nq}):
            n = nk - nq + r + 1 if causal else nk
            for head in (0, q_heads - 1):
                at = slice(j, j + n), slice(head // (q_heads // 2), head // (q_heads // 2) + 1)
                one = slice(i + r, i + r + 1), slice(head, head + 1)
                want, tol = attend64(f64(q[one]), f64(k[at]), f64(clean[at]), dim ** -0.5, False)
                with np.errstate(invalid="ignore"):
                    if head == 0:
                        for column, odd in part[3].items():
                            seen = [x for place, x in odd if place < n]
                            want[0, 0, column] = _sum_of(seen) if seen else want[0, 0, column]
                    within(got[one], want, tol, f"query {r} of {nq} on {nk}, head {head}")
                same = np.isinf(want)
                assert np.array_equal(np.isnan(want), np.isnan(got[one])) and np.array_equal(got[one][same], want[same])
        i, j = i + nq, j + nk


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [64, 128, 96])
@pytest.mark.parametrize("n,q_heads", [(40, 4), (900, 16), (1100, 64)])
def test_prompt_of_infinite_keys(dev, rng, n, q_heads, dim, causal):
    """A key with an infinity scores +inf (NaN) or -inf (not there), by the sign of the query's value."""
    q, k, v = normal(rng, n, q_heads, dim), normal(rng, n, 2, dim), normal(rng, n, 2, dim)
    place = n // 3
    k[place, 0, 3] = np.inf
    q[:, :, 3] = np.where(np.arange(n) % 2, 1, -1)[:, None]
    got = Prompt(dev, q, k, v, [n], [n], causal, dim ** -0.5).run()
    for r in (0, place - 1, place, place + 1, n - 2, n - 1):
        seen = np.arange(r + 1 if causal else n)
        rest = seen[seen != place]
        for head in (0, q_heads - 1):
            first = head < q_heads // 2
            kv = slice(0, 1) if first else slice(1, 2)
            use = rest if first else seen
            want, tol = attend64(f64(q[r:r + 1, head:head + 1]), f64(k[use, kv]), f64(v[use, kv]), dim ** -0.5, False)
            if first and place in seen and r % 2:
                want[:] = np.nan
            with np.errstate(invalid="ignore"):
                within(got[r:r + 1, head:head + 1], want, tol, f"query {r}, head {head}")


# ------------------------------------------------------------ many short sequences

@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("sequences,heads,most", [(65, 1, 1), (100, 2, 5), (70, 3, 32), (130, 8, 64), (200, 6, 128)])
def test_prompt_many_sequences_of_one_tile(dev, rng, sequences, heads, most, dim, causal):
    """More sequences than a wave has lanes that fit a tile each, empty ones among them, on more keys."""
    queries = [int(n) for n in rng.integers(0, most + 1, sequences)]
    queries[3], queries[sequences - 1] = most, 1
    keys = [n + int(more) for n, more in zip(queries, rng.choice([0, 1, 60, 200], sequences))]
    q = normal(rng, sum(queries), heads, dim)
    k, v = normal(rng, sum(keys), 1, dim), normal(rng, sum(keys), 1, dim)
    got = Prompt(dev, q, k, v, queries, keys, causal, dim ** -0.5).run()
    i = j = 0
    for nq, nk in zip(queries, keys):
        a, b = slice(i, i + nq), slice(j, j + nk)
        want, tol = attend64(f64(q[a, -1:]), f64(k[b]), f64(v[b]), dim ** -0.5, causal)
        within(got[a, -1:], want, tol, f"{nq} on {nk}") if nq else None
        i, j = i + nq, j + nk
    assert np.isfinite(got).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 24])
def test_tokens_of_lengths_at_31_bits(dev, rng, kind, dim):
    """Contexts that end at 2^31 - 1 tokens and a little before it, on one page of zero keys that repeats and a last
    one with two keys that weigh e^40 times the others: what 2^31 of those add is below 2^-25."""
    last, page, width = (1 << 31) - 1, 1 << 16, 1 << 15
    cache = Cache(dev, kind, 2, page, 1, dim)
    k, v = np.zeros((page, 1, dim), np.float16), rng.standard_normal((page, 1, dim)).astype(np.float16)
    cache.write(k, v, np.arange(page))
    k[[-22, -2], 0, 0] = 40                 # places last - 21 and last - 1
    cache.write(k[:-1], v[:-1], np.arange(page, 2 * page - 1))
    table = np.zeros((3, width), np.int32)
    table[:, -1] = 1
    q = np.zeros((3, 2, dim), np.float16)
    q[..., 0] = 1
    got = Token(cache, q, table, [last, last - 20, 40], 1.0).run()
    sv = stored64(v, kind)[:, 0]
    for stream, (want, size) in enumerate((((sv[-22] + sv[-2]) / 2, np.maximum(abs(sv[-22]), abs(sv[-2]))), (sv[-22], abs(sv[-22])),
                                           (sv[:40].mean(0), np.abs(sv[:40]).max(0)))):
        # The weights' rounding and the output's, and the other tokens.
        within(got[stream], np.broadcast_to(want, (2, dim)), size * 2.0 ** -10 + 2.0 ** -20, f"stream {stream}")
