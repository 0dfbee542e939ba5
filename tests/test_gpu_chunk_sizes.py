"""nnhip_attn_chunk and nnhip_attn_chunk8: keys and queries of any size that float32 holds, whose scores are a few units."""
import math

import numpy as np
import pytest

import chunk_helpers as ch
from test_gpu_chunk import cache_for, check_chunk, run_chunk

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("new,past,dim", [(4, 100, 64), (9, 60, 30), (40, 300, 64), (140, 300, 128), (6, 2000, 128)])
@pytest.mark.parametrize("k_size,alpha", [(1e37, 0.3), (1e35, -0.3), (1e32, 0.3), (1e29, 0.3), (1e25, 0.3), (1e22, 0.3), (1e-30, 0.3), (1e-37, 0.3),
                                          (1e-37, 3e4)])
def test_sizes_of_keys(k_size, alpha, new, past, dim, slopes, bits):
    """Each row of the cache of a size of its own, within 2^-6 to 1 of k_size; every fifth one ordinary."""
    rng = np.random.default_rng(new)
    page, heads, per = 16, 1, 2
    lens, start = [new + past], [0, new]
    x, table, pages = cache_for(rng, lens, page, heads, dim, bits)
    size = (2.0 ** rng.integers(-6, 1, len(x["K"])) * k_size).astype(np.float32)
    size[::5] = 1
    if bits == 32:
        x["K"] = x["K"] * size[:, None, None]
        x["K64"] = x["K"].astype(np.float64)
    else:
        x["Ks"] = x["Ks"] * size[:, None]
        x["K64"] = x["K"].astype(np.float64) * x["Ks"].astype(np.float64)[..., None]
    q = (rng.normal(size=(new, per, dim)) / k_size).clip(-1e37, 1e37).astype(np.float32)
    if k_size < 1:             # ordinary rows would have scores past float32
        for j in range(lens[0]):
            r = ch.row_of(table, 0, j, page, pages)
            if size[r] == 1:
                x["K"][r], x["K64"][r] = 0, 0
    alpha = np.float32(alpha)
    sl = np.array([0.25, 0.01], np.float32) if slopes else None
    c = dict(pages=pages, page=page, heads=heads, dim=dim)
    got = run_chunk(x, c, table, q, start, new, lens, sl, alpha)
    want = ch.attend(q, x["K64"], x["V64"], table, page, pages, heads, start, new, lens, float(alpha), sl)
    check_chunk(got, want)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("new,past,dim", [(4, 100, 64), (9, 60, 30), (40, 300, 64), (140, 300, 128), (6, 2000, 128)])
def test_one_large_key_of_negative_scores(new, past, dim, bits):
    """One key of 4e36 whose scores are -1.2, among others of 0: nothing says that a product left float32's range but a
    weight that is missing."""
    rng = np.random.default_rng(new)
    page, heads = 16, 1
    lens, start = [new + past], [0, new]
    x, table, pages = cache_for(rng, lens, page, heads, dim, bits)
    r = ch.row_of(table, 0, past // 2, page, pages)
    x["K"][...] = 0
    if bits == 32:
        x["K"][r, :, 0] = -4e36
        x["K64"] = x["K"].astype(np.float64)
    else:
        x["K"][r, :, 0] = -127
        x["Ks"][r] = 4e36 / 127
        x["K64"] = x["K"].astype(np.float64) * np.where(np.isfinite(x["Ks"]), x["Ks"], 0).astype(np.float64)[..., None]
    q = np.zeros((new, 2, dim), np.float32)
    q[..., 0] = 1e-36
    c = dict(pages=pages, page=page, heads=heads, dim=dim)
    got = run_chunk(x, c, table, q, start, new, lens, None, np.float32(0.3))
    check_chunk(got, ch.attend(q, x["K64"], x["V64"], table, page, pages, heads, start, new, lens, float(np.float32(0.3))))
    others = past + np.arange(new)[:, None]   # their weights are 1 each, and sums of ones exact
    assert np.all(np.abs(got[2] - others - math.exp(-1.2)) < 2.0 ** -10)
