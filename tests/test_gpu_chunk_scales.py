"""nnhip_attn_chunk8: a row that sees a scale that is not finite is NaN, whatever weight that position has, on every route
(up to 16, up to 32 and more rows of a key head, rows that are read in pieces and byte by byte, one and several ranges)."""
import numpy as np
import pytest

import chunk_helpers as ch
import test_chunk_scales as cpu_tests
from test_gpu_chunk import cache_for, run_chunk

pytestmark = pytest.mark.gpu

ROUTES = [(9, 20, 1, 64), (5, 0, 4, 30), (20, 3, 1, 48), (40, 100, 1, 64), (70, 10, 2, 128), (200, 33, 1, 96), (40, 20, 2, 17),
          (3, 1500, 4, 128), (150, 900, 1, 40)]


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("which", ["Vs", "Ks"])
@pytest.mark.parametrize("new,past,per,dim", ROUTES)
def test_under_a_weight_of_nothing(new, past, per, dim, which, value):
    """Position 0 has a score of 900, every other one far below: their weights underflow to 0. The scale that is not finite
    lies in the same tile as position 0, in later ones, and at the last position but one."""
    rng = np.random.default_rng(new + dim)
    page, heads, n = 16, 2, new + past
    lens, start = [n], [0, new]
    x, table, pages = cache_for(rng, lens, page, heads, dim, 8)
    q = rng.normal(size=(new, heads * per, dim)).astype(np.float32)
    q[..., 0] = 8
    rows = [ch.row_of(table, 0, j, page, pages) for j in range(n)]
    x["K"][rows, :, 0] = -1
    x["K"][rows[0], :] = 0
    x["K"][rows[0], :, 0] = 127
    x["Ks"][rows[0]] = 900 / 127
    x["K64"] = x["K"].astype(np.float64) * x["Ks"].astype(np.float64)[..., None]
    c = dict(pages=pages, page=page, heads=heads, dim=dim)
    want = ch.attend(q, x["K64"], x["V64"], table, page, pages, heads, start, new, lens, 0.125)
    for at in sorted({min(5, n - 1), n // 2, n - 2}):
        y = {k: a.copy() for k, a in x.items()}
        y[which][rows[at], 0] = value
        if which == "Ks":      # one sign of the query's product throughout: a score of -inf by the formula, not NaN
            y["K"][rows[at], 0] = 0
            y["K"][rows[at], 0, 0] = -127 if value > 0 else 127
        O, m, l = run_chunk(y, c, table, q, start, new, lens, None, 0.125)
        first = max(0, at - past)
        assert np.isnan(O[first:, :per]).all(), (at, np.argwhere(~np.isnan(O[first:, :per]))[:3])
        assert np.all(np.abs(O[:first] - want[0][:first]) <= want[3][:first])
        assert np.all(np.abs(O[:, per:] - want[0][:, per:]) <= want[3][:, per:])


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("at", [1, 3, 5])
def test_rows_not_finite(hip, which, at):
    cpu_tests.rows_not_finite(hip, which, at)


@pytest.mark.parametrize("bits", [32, 8])
def test_queries_not_finite(hip, bits):
    cpu_tests.queries_not_finite(hip, bits)
