"""nnhip_attn_paged over positions that several ranges, waves and walks take (csrc/k_attn_paged.hip), against the 64-bit
form (paged_helpers.attend): what must not depend on how a call is cut."""
import numpy as np
import pytest

import paged_helpers as ph
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
