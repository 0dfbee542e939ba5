"""nnhip_attn_paged over positions that several ranges, waves and walks take (csrc/k_attn_paged.hip), against the 64-bit
form (paged_helpers.attend): what must not depend on how a call is cut."""
import math

import numpy as np
import pytest

import paged_helpers as ph
import test_gpu_paged as tp
from test_gpu_paged import run_attend

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("beams,n,shared,dim", [(1, 60, None, 64), (1, 700, None, 64), (1, 2000, None, 80), (3, 700, [640.0], 64),
                                                (3, 2000, [1984.0], 20), (40, 700, [640.0], 64), (40, 9000, [8960.0], 32),
                                                (3, 700, [0.0], 64)])
def test_value_not_finite_under_a_small_weight(beams, n, shared, dim, value):
    """A value that is not finite makes O so, however small its weight and wherever the ranges end: the scores of the
    first 64 positions are 200 below the others'."""
    rng = np.random.default_rng(n + beams)
    page = 16
    pages = -(-n // page)
    K, V = (rng.normal(size=(pages * page, 1, dim)).astype(np.float32) for _ in range(2))
    K[:64, 0, 0] -= 200.0
    V[10, 0, 5] = value
    q = (rng.normal(size=(beams, 1, dim)) * 0.1).astype(np.float32)
    q[:, 0, 0] = 1.0
    table = np.tile(np.arange(pages, dtype=np.float32), (beams, 1))
    c = dict(pages=pages, page=page, heads=1, dim=dim)
    lens = [n] * beams
    O, _, _ = run_attend(c, q, K, V, table, lens, shared, beams, None, 1.0)
    wO, _, _, tol = ph.attend(q, K, V, table, page, pages, 1, lens, 1.0)
    assert not np.isfinite(wO[:, 0, 5]).any() and not np.isfinite(O[:, 0, 5]).any()
    rest = np.arange(dim) != 5
    assert np.all(np.abs(O[:, 0, rest] - wO[:, 0, rest]) <= tol[:, 0, rest])


@pytest.mark.parametrize("beams,first,dim,per", [(4, 1, 64, 1), (4, 3, 30, 2), (40, 7, 64, 1), (140, 130, 32, 1), (9, 2, 128, 4)])
@pytest.mark.parametrize("short", [0, 5, 95])
def test_group_whose_first_sequences_are_short(beams, first, dim, per, short):
    """The shared positions are read through the first sequence that has them all, whatever the tables of the shorter ones
    in front of it name there; where no sequence has them all each is read through its own table."""
    rng = np.random.default_rng(beams + dim)
    page, width, n = 16, 8, 96
    table = np.tile(rng.permutation(60)[:width].astype(np.float32), (beams, 1))
    table[:first] = -1.0
    table[:first, :short // page + 1] = 60 + np.arange(short // page + 1)     # rows of their own
    table[1::2, 6:] = [[70, 71]]
    K, V = (rng.normal(size=(80 * page, 1, dim)).astype(np.float32) for _ in range(2))
    q = rng.normal(size=(beams, per, dim)).astype(np.float32)
    lens = np.array([short] * first + [n + int(x) for x in rng.integers(0, 20, beams - first)], np.float32)
    c = dict(pages=80, page=page, heads=1, dim=dim)
    for ls in (lens, np.minimum(lens, 95)):
        O, m, l = run_attend(c, q, K, V, table, ls, [float(n)], beams, None, 0.125)
        wO, wm, wl, tol = ph.attend(q, K, V, table, page, 80, 1, ls, 0.125)
        assert np.all(np.abs(O - wO) <= tol)


def two_positions(rows, dim):
    """A group of `rows` sequences that share 64 positions, all absent but two of one tile: queries, caches, table, lengths."""
    q = np.zeros((rows, 1, dim), np.float32)
    K, V = np.zeros((64, 1, dim), np.float32), np.zeros((64, 1, dim), np.float32)
    table = np.full((rows, 64), -1.0, np.float32)
    table[:, 3], table[:, 9] = 3, 9
    return q, K, V, table, [64] * rows, dict(pages=64, page=1, heads=1, dim=dim)


@pytest.mark.parametrize("rows,dim", [(12, 64), (32, 64), (40, 64), (64, 128), (130, 32)])
def test_weight_to_its_last_bits(rows, dim):
    """Scores 0 and -x, values 0 and 1: O = z / (1 + z), z = exp(-x), 0.69 < x < 1.39. Score, products and sums are exact (one
    factor has one bit); the exponent's argument, below 2, is off by its rounding, 2^-24, and log2(e)'s, 2^-25.1, times
    ln 2, exp2 by a unit in its last place, 2^-23 of z, together 3.1 2^-24 of z and, times 1 / (1 + z) <= 0.8, 2.5 2^-24 of O;
    1 + z and the quotient round once each, 2^-24: 4.5 2^-24 of O. The x are those at which an argument near 24 would round
    by nearly 2^-20, 16 times as far."""
    rng = np.random.default_rng(rows)
    q, K, V, table, lens, c = two_positions(rows, dim)
    x = rng.uniform(0.7, 1.38, 20000).astype(np.float32)
    half = np.abs((24 - x.astype(np.float64) / np.log(2)) * 2.0 ** 19 % 1 - 0.5)
    x = x[np.argsort(half)[:rows]]
    q[:, 0, 1], K[9, 0, 1], V[9, 0] = -x, 1, 2.0 ** rng.integers(-3, 4, dim)
    O, m, l = run_attend(c, q, K, V, table, lens, [64.0], rows, None, 1.0)
    z = np.exp(-x.astype(np.float64))
    assert np.all(m == 0) and np.all(np.abs(l[:, 0] - (1 + z)) <= (3.1 * z + 1.5) * U)
    want = (z / (1 + z))[:, None] * V[9, 0].astype(np.float64)
    assert np.all(np.abs(O[:, 0] - want) <= 4.5 * U * np.abs(want))


@pytest.mark.parametrize("rows,dim", [(12, 64), (40, 64), (64, 128), (130, 32)])
def test_every_part_of_the_products(rows, dim):
    """As above with factors of 24 bits. A product of three bf16 parts each leaves out (2^-24 + 2^-34) of itself, and its
    six terms' sum, smallest first, is rounded or cut, 2^-23 for the last addition and 5 2^-31 before: 3.1 2^-24. A score of
    up to 1.39 is off by 4.4 2^-24, with the argument's and exp2's 3.1 2^-24 z by 7.5 2^-24, O by 0.8 times that, by 3.1 2^-24
    for its own product and 2 2^-24 for 1 + z and the quotient: 11.1 2^-24. A third part left out anywhere is up to 2^-16."""
    rng = np.random.default_rng(rows + 1)
    q, K, V, table, lens, c = two_positions(rows, dim)
    K[9, 0, 1] = np.float32(rng.uniform(1.2, 1.3))
    q[:, 0, 1] = -rng.uniform(0.6, 1.06, rows)
    V[9, 0] = rng.normal(size=dim)
    O, m, l = run_attend(c, q, K, V, table, lens, [64.0], rows, None, 1.0)
    z = np.exp(q[:, 0, 1].astype(np.float64) * float(K[9, 0, 1]))
    assert z.max() < 0.5 and z.min() > 0.25
    want = (z / (1 + z))[:, None] * V[9, 0].astype(np.float64)
    assert np.all(np.abs(O[:, 0] - want) <= 11.1 * U * np.abs(want))
    assert np.all(np.abs(l[:, 0] - (1 + z)) <= (7.5 * z + 1.5) * U)


@pytest.mark.parametrize("size", [1100, 1250, 1340, 1360, 1380, 1400, 1420, 1450])
def test_small_values_under_growing_scores(size):
    """Values of 2^-100 under scores that grow by 69 to 91 over each of 16 ranges: neither the weights nor the products
    overflow where the factor to the largest score is below every normal float."""
    rng = np.random.default_rng(size)
    heads, per, beams, dim, n, page = 16, 4, 10, 32, 8000, 16
    lens = [n + int(x) for x in rng.integers(1, 9, beams)]
    table, pages = tp.batch_of(rng, 1, beams, page, [n], lens, True)
    K = (rng.normal(size=(pages * page, heads, dim)) * 0.1).astype(np.float32)
    V = (rng.normal(size=(pages * page, heads, dim)) * 2.0 ** -100).astype(np.float32)
    q = (rng.normal(size=(beams, heads * per, dim)) * 0.25).astype(np.float32)
    q[:, :, 0] = 1.0
    rows = [ph.row_of(table, 0, j, page, pages) for j in range(n)]
    K[rows, :, 0] = np.linspace(0, size, n).astype(np.float32)[:, None]
    c = dict(pages=pages, page=page, heads=heads, dim=dim)
    O, m, l = run_attend(c, q, K, V, table, lens, [n], beams, None, 1.0)
    wO, wm, wl, tol = ph.attend(q, K, V, table, page, pages, heads, lens, 1.0)
    assert np.all(np.abs(O - wO) <= tol) and np.all(np.abs(wO).max(axis=2) > 2.0 ** -110)


def check_stats(c, q, K, V, table, lens, shared, alpha, slopes=None):
    """test_gpu_paged.check_many, and m and l: a score is off by what its products, the slope's and the sums round, l by
    what its weights and their sum are (as in test_attend); without a position they are lowest() and 0."""
    beams, dim = q.shape[0], q.shape[2]
    O, m, l = run_attend(c, q, K, V, table, lens, shared, beams, slopes, alpha)
    wO, wm, wl, tol = ph.attend(q, K, V, table, c["page"], c["pages"], 1, lens, alpha, slopes)
    ok = np.isfinite(wO)
    assert np.array_equal(np.isfinite(O), ok) and np.all(np.abs(O[ok] - wO[ok]) <= tol[ok])
    fin = np.isfinite(wl)
    assert np.array_equal(np.isfinite(l), fin)
    size = np.zeros(wm.shape)
    for b in range(beams):
        rows = [ph.row_of(table, b, j, c["page"], c["pages"]) for j in range(ph.length_of(lens[b], table.shape[1] * c["page"]))]
        k = np.abs(K[[r for r in rows if r is not None], 0].astype(np.float64))
        if len(k):
            with np.errstate(invalid="ignore"):
                size[b] = abs(alpha) * (k @ np.abs(q[b].astype(np.float64)).T).max(axis=0)
    s_tol = (dim + 8) * U * size + 8 * U * np.abs(wm)
    if slopes is not None:
        s_tol = s_tol + 2 * U * np.abs(slopes)[None, :] * max(lens)
    n = max(lens)
    assert np.all(np.abs(m[fin] - wm[fin]) <= s_tol[fin])
    assert np.all(np.abs(l[fin] - wl[fin]) <= wl[fin] * (4 * s_tol[fin] + 2 * n * U))
    none = wl == 0
    assert np.all(l[none] == 0) and np.all(m[none] == np.float32(-3.4028234663852886e38))
    return O


@pytest.mark.parametrize("beams,per,dim,prefix,own", [(9, 4, 32, 130, 20), (33, 1, 64, 400, 9), (40, 3, 96, 700, 5),
                                                     (16, 4, 128, 1500, 40), (70, 2, 128, 333, 3), (40, 1, 80, 200, 7),
                                                     (3, 20, 128, 200, 50)])
@pytest.mark.parametrize("slopes", [False, True])
def test_many_rows_m_and_l(beams, per, dim, prefix, own, slopes):
    """The bf16 walk's m and l: also of a sequence shorter than the shared positions, of one of length 0, beside rows past
    the last one."""
    rng = np.random.default_rng(beams * 100 + dim + 1)
    c, q, K, V, table, lens, shared = tp.many_rows(rng, beams, per, dim, prefix, own)
    tp.poison(K, V, table, lens, c["page"], c["pages"])
    lens[1] = shared[0] - 3
    lens[2] = 0
    sl = (2.0 ** -np.arange(3, per + 3)).astype(np.float32) if slopes else None
    O = check_stats(c, q, K, V, table, lens, shared, 1 / math.sqrt(dim), sl)
    assert np.all(O[2] == 0)


@pytest.mark.parametrize("what", tp.test_attend_many_rows_range.pytestmark[0].args[1])
def test_many_rows_range_m_and_l(what, monkeypatch):
    """The same where the bf16 parts do not hold the values and the range is walked again."""
    monkeypatch.setattr(tp, "check_many", check_stats)
    tp.test_attend_many_rows_range(what)
