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
