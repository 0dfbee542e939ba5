"""nnhip_attn_chunk and nnhip_attn_chunk8: large values under small weights take no accuracy from the others, however many
rows a sequence has."""
import numpy as np
import pytest

import chunk_helpers as ch
from test_gpu_chunk import cache_for, run_chunk

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def check(O, q, x, rows, past, per, alpha):
    """One sequence whose positions lie in these rows. Scores, weights and their products with the values as
    chunk_helpers.attend bounds them, but for the parts: what is below 2^-39 of the row's largest product of a weight and a
    value is lost. Products are held against twice the largest of them at most, and a value against twice its row's
    largest, and where weights shrink on the way against another two: 2^-36 of the largest, for each position."""
    N, H, D = q.shape
    for i in range(N):
        r = rows[:past + i + 1]
        for h in range(H):
            K, V, z = x["K64"][r, h // per], x["V64"][r, h // per], q[i, h].astype(np.float64)
            s = alpha * (K @ z)
            size = abs(alpha) * (np.abs(K) @ np.abs(z) * (1 + 7 * 2.0 ** -24) + D * 2.0 ** -14 * np.abs(K).max(1) * np.abs(z).max())
            w = np.exp(s - s.max())
            w /= w.sum()
            off = 2 * ((D + 7) * U * size.max() + 4 * U * np.abs(s).max() + 4 * U) + (2 * len(r) + 3) * U
            tol = 2 * off * (w @ np.abs(V)) + len(r) * 2.0 ** -36 * (w * np.abs(V).max(1)).max() + 1e-30
            bad = ~(np.abs(O[i, h] - w @ V) <= tol)
            assert not bad.any(), (i, h, O[i, h][bad][:4], (w @ V)[bad][:4], tol[bad][:4])


def put_key(x, rows, score):
    """Keys of rows that give these scores with queries of 8 in feature 0 and alpha 1 / 8."""
    score = np.asarray(score, np.float32)
    x["K"][rows] = 0
    if "Ks" in x:
        x["K"][rows, :, 0] = (np.sign(score) * 127).astype(np.int8)[:, None]
        x["Ks"][rows] = (np.maximum(np.abs(score), np.float32(1e-3)) / 127)[:, None]
        x["K64"][rows] = x["K"][rows].astype(np.float64) * x["Ks"][rows].astype(np.float64)[..., None]
    else:
        x["K"][rows, :, 0] = score[:, None]
        x["K64"][rows] = x["K"][rows]


def grow(x, row, by):
    if "Vs" in x:
        x["Vs"][row] *= np.float32(by)
        x["V64"][row] = x["V"][row].astype(np.float64) * x["Vs"][row].astype(np.float64)[:, None]
    else:
        x["V"][row] *= np.float32(by)
        x["V64"][row] = x["V"][row]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("new,past,per,dim", [(9, 20, 1, 64), (5, 0, 4, 30), (20, 3, 1, 48), (40, 100, 1, 64), (70, 10, 2, 128), (200, 33, 1, 96),
                                              (3, 1500, 4, 128), (150, 900, 1, 40), (40, 20, 2, 17)])
def test_a_large_value_under_a_small_weight(new, past, per, dim, bits):
    """A value of 1e12 (1e30) under a weight of e^-60 (e^-110) of the others': what it adds to the sum is nothing."""
    rng = np.random.default_rng(new + dim)
    page, heads, n = 16, 2, new + past
    for size, score in ((1e12, -60.0), (1e30, -110.0)):
        for at in sorted({0, n // 2}):
            x, table, pages = cache_for(rng, [n], page, heads, dim, bits)
            rows = np.array([ch.row_of(table, 0, j, page, pages) for j in range(n)])
            q = rng.normal(size=(new, heads * per, dim)).astype(np.float32)
            q[..., 0] = 8
            x["K"][rows, :, 0] = 0
            x["K64"][rows, :, 0] = 0
            put_key(x, rows[at:at + 1], [score])
            grow(x, rows[at], size)
            c = dict(pages=pages, page=page, heads=heads, dim=dim)
            O, _, _ = run_chunk(x, c, table, q, [0, new], new, [n], None, 0.125)
            first = 0 if at else 1   # a token that sees the large value alone has it
            check(O[first:], q[first:], x, rows, past + first, per, 0.125)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("new,per", [(2, 1), (6, 4), (40, 1)])
def test_a_large_value_that_is_outgrown(new, per, bits):
    """Scores that rise by less than one bit a tile of 32 positions, up to e^90 above the first, whose value is 1e25; and by
    hundreds at once behind it."""
    rng = np.random.default_rng(new)
    page, heads, dim, n = 64, 1, 64, 6000
    x, table, pages = cache_for(rng, [n], page, heads, dim, bits)
    rows = np.array([ch.row_of(table, 0, j, page, pages) for j in range(n)])
    q = rng.normal(size=(new, per, dim)).astype(np.float32)
    q[..., 0] = 8
    c = dict(pages=pages, page=page, heads=heads, dim=dim)
    grow(x, rows[0], 1e25)
    for score in (np.arange(n) * 0.015, np.where(np.arange(n) < n // 2, 0.0, 300.0), np.where(np.arange(n) < n - new, 0.0, 90.0)):
        put_key(x, rows, score)
        O, _, _ = run_chunk(x, c, table, q, [0, new], new, [n], None, 0.125)
        check(O, q, x, rows, n - new, per, 0.125)
