"""nnhip_attn_chunk with up to 32 rows of a key head: float32 products throughout, so that features of very different sizes
are as exact as each other."""
import numpy as np
import pytest

import chunk_helpers as ch
from test_gpu_chunk import cache_for, run_chunk

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("new,past,per,dim,page", [([4, 1], [100, 700], 1, 64, 16), ([5], [60], 4, 30, 8), ([20, 3], [3, 900], 1, 48, 16),
                                                   ([8, 1], [2000, 4], 4, 128, 64), ([1] * 40, list(range(40)), 2, 96, 16)])
def test_features_of_many_sizes(new, past, per, dim, page):
    """Features of keys and values of sizes from 1e-12 to 1e12, queries' the other way round. A score is off by a chain of
    products and additions, (dim + 4) 2^-24 of its terms' sizes, its exponent's argument by 4 2^-24 of the scores' and exp2
    by as much, a sum over n weights by n 2^-24 more, numerator and denominator alike; of no feature by another's size."""
    rng = np.random.default_rng(dim)
    heads = 2
    lens, start = [n + p for n, p in zip(new, past)], np.concatenate([[0], np.cumsum(new)])
    x, table, pages = cache_for(rng, lens, page, heads, dim, 32)
    size = (10.0 ** rng.uniform(-12, 12, dim)).astype(np.float32)
    x["K"], x["V"] = x["K"] * size, x["V"] * size
    q = (rng.normal(size=(int(start[-1]), heads * per, dim)) / size).astype(np.float32)
    O, m, l = run_chunk(x, dict(pages=pages, page=page, heads=heads, dim=dim), table, q, start, max(new), lens, None, 0.125)
    for b, n in enumerate(new):
        rows = np.array([ch.row_of(table, b, j, page, pages) for j in range(lens[b])])
        for i in range(n):
            r, t = rows[:lens[b] - n + i + 1], start[b] + i
            for h in range(heads * per):
                K, V, z = x["K"][r, h // per].astype(np.float64), x["V"][r, h // per].astype(np.float64), q[t, h].astype(np.float64)
                s = 0.125 * (K @ z)
                w = np.exp(s - s.max())
                w /= w.sum()
                score = (dim + 4) * U * (0.125 * (np.abs(K) @ np.abs(z))).max() + 4 * U * np.abs(s).max() + 4 * U
                tol = 2 * (2 * score + (2 * len(r) + 3) * U) * (w @ np.abs(V))
                bad = ~(np.abs(O[t, h] - w @ V) <= tol)
                assert not bad.any(), (t, h, O[t, h][bad][:4], (w @ V)[bad][:4], tol[bad][:4])
