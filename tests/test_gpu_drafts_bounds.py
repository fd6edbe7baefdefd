"""Drafts where a context, a list or a number ends: cuts, drafts that do not
count, pages that ran out, the last lengths and the largest scores."""

import numpy as np
import pytest

from devmem import Dev
from drafts import Contexts, Drafts, drafts_seen, masked64, tops_of, tree
from mlvc_hip import KV_E4M3, KV_F16, KV_INT8
from tokens import Cache, f64, stored64, within

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
