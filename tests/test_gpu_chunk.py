"""8-bit caches, attention of chunks of new tokens and draft verification (include/nnhip_kernels.h: nnhip_kv8_append,
nnhip_kv8_read, nnhip_attn_chunk, nnhip_attn_chunk8, nnhip_draft_verify) against plain 64-bit forms (chunk_helpers.py).

Every buffer's untouched parts are checked as well: rows of the caches that no token names, the gaps of strided outputs,
padding. Rows that must not be read hold NaN.
"""
import math

import numpy as np
import pytest
import torch

import chunk_helpers as ch
from test_gpu_paged import dev, layout, ptr, stream

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def dev8(a):
    return torch.as_tensor(np.ascontiguousarray(a, dtype=np.int8)).cuda()


def pages_of(c, K, V, table, Ks=None, Vs=None):
    sizes = (table.shape[0], table.shape[1], c["pages"], c["page"], c["heads"], c["dim"], c.get("row", c["heads"] * c["dim"]))
    if Ks is None:
        return ch.Pages(ptr(K), ptr(V), ptr(table), *sizes)
    return ch.Pages8(ptr(K), ptr(V), ptr(Ks), ptr(Vs), ptr(table), *sizes)


# -- 8-bit caches ----------------------------------------------------------------
STORE = [  # tokens, batch, q_heads, heads, dim, rope, page, layout, seq
    (1, 1, 1, 1, 1, 0, 1, "token", True),
    (4, 4, 12, 12, 64, 64, 1, "feature", False),
    (3, 2, 2, 1, 2, 2, 3, "token", True),
    (33, 5, 8, 2, 128, 128, 16, "token", True),
    (70, 3, 6, 6, 80, 40, 64, "feature", True),
    (70, 3, 6, 6, 80, 40, 64, "token", True),
    (65, 7, 3, 3, 30, 28, 24, "gaps", True),
    (50, 2, 4, 2, 17, 6, 8, "strided", True),
    (40, 3, 2, 2, 256, 256, 16, "token", True),
    (41, 3, 2, 2, 248, 16, 16, "token", True),
    (129, 1, 4, 4, 36, 36, 7, "feature", True),
    (9, 9, 0, 4, 64, 64, 16, "feature", False),
    (300, 4, 8, 4, 96, 0, 16, "token", True),
    (77, 4, 5, 5, 12, 8, 16, "token", True),
]


@pytest.mark.parametrize("tokens,batch,q_heads,heads,dim,rope,page,kind,with_seq", STORE)
def test_store_and_read(tokens, batch, q_heads, heads, dim, rope, page, kind, with_seq):
    rng = np.random.default_rng(tokens * 131 + dim)
    per = -(-tokens // batch) + 5
    width = -(-per // page) + 1
    pages = batch * width + 2
    f = heads * dim
    row = f + (5 if kind == "gaps" else 0)
    c = dict(pages=pages, page=page, heads=heads, dim=dim, row=row)
    table = rng.permutation(pages)[:batch * width].reshape(batch, width).astype(np.float32)
    if with_seq:
        order = rng.permutation(batch * per)[:tokens]
        seq, pos = order // per, (order % per).astype(np.float32)
    else:
        seq, pos = np.arange(tokens), rng.integers(0, per, tokens).astype(np.float32)
    rope_rows = per - 2
    seq = seq.astype(np.float32)
    if tokens >= 30:           # padding: no position, no sequence, no page, no row of the rotation
        pos[3], pos[5], pos[7], pos[11] = -1, np.nan, width * page, 2.0 ** 30
        table[0, 0], table[batch - 1, width - 1] = -1, np.nan
        table[batch // 2, 0] = pages
        seq[13], seq[17], seq[19] = -1, batch, np.nan
    k, v = (rng.normal(size=(tokens, f)).astype(np.float32) for _ in range(2))
    if tokens >= 30:           # rows of zeros, of the smallest and largest floats, values that are not finite, exact ties
        k[0], k[1, :dim], k[2, :dim], k[4, 0] = 0, 1e-45, 3e38, np.inf
        v[0], v[1, :dim], v[2, :dim], v[4, 0], v[6, f - 1] = 0, 2e-44, -3e38, np.nan, -np.inf
        v[8, :dim] = (np.arange(dim) % 250 - 124.5) * 3
        v[8, 0] = 127 * 3
    q = rng.normal(size=(tokens, max(1, q_heads) * dim)).astype(np.float32)
    ang = rng.uniform(-3, 3, (rope_rows, max(1, rope // 2)))
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    K0, V0 = (rng.integers(-127, 128, (pages * page, row)).astype(np.int8) for _ in range(2))
    Ks0, Vs0 = (rng.uniform(0.1, 1, (pages * page, heads)).astype(np.float32) for _ in range(2))
    (tk, sk, _), (tv, sv, _), (tq, sq, _) = (layout(x, kind, rng) for x in (k, v, q))
    out0 = np.full_like(q, 5.0)
    to, so, read_o = layout(out0, "feature" if kind == "token" and dim < 100 else kind, rng)
    K, V, Ks, Vs, tt, tc, tsn = dev8(K0), dev8(V0), dev(Ks0), dev(Vs0), dev(table), dev(cos), dev(sin)
    tseq, tpos = dev(seq), dev(pos)
    pg = pages_of(c, K, V, tt, Ks, Vs)
    print(f"[store] {tokens} tokens heads {heads} dim {dim} rope {rope} page {page} {kind}", flush=True)
    lib = ch.library()
    assert lib.nnhip_kv8_append(
        pg, ptr(tk), *sk, ptr(tv), *sv, ptr(tq) if q_heads else None, *sq, ptr(to) if q_heads else None, *so, q_heads, tokens,
        ptr(tseq) if with_seq else None, ptr(tpos), ptr(tc) if rope else None, ptr(tsn) if rope else None,
        rope_rows if rope else 0, rope, stream()) == 0
    wK, wV, wKs, wVs, wo, tol = K0.copy(), V0.copy(), Ks0.copy(), Vs0.copy(), out0.astype(np.float64), np.zeros(out0.shape)
    h = rope // 2
    for n in range(tokens):
        r, p = ch.place(table, batch, page, pages, seq if with_seq else None, pos, rope_rows if rope else 0, n)
        if r is None:
            continue
        co, si = (cos[p], sin[p]) if rope else (None, None)
        by, wKs[r] = ch.quantise(ch.turned(k[n].reshape(heads, dim), co, si, rope))
        wK[r, :f] = by.reshape(-1)
        by, wVs[r] = ch.quantise(v[n].reshape(heads, dim).astype(np.float64))
        wV[r, :f] = by.reshape(-1)
        if q_heads:
            x = q[n].reshape(q_heads, dim)
            wo[n] = ch.turned(x, co, si, rope).reshape(-1)
            size = np.zeros((q_heads, dim))
            if h:
                a, b = np.abs(x[:, :h]), np.abs(x[:, h:2 * h])
                size[:, :h], size[:, h:2 * h] = a * abs(co) + b * abs(si), b * abs(co) + a * abs(si)
            tol[n] = 2 * U * size.reshape(-1)
    assert np.array_equal(Ks.cpu().numpy(), wKs, equal_nan=True) and np.array_equal(Vs.cpu().numpy(), wVs, equal_nan=True)
    assert np.array_equal(K.cpu().numpy(), wK) and np.array_equal(V.cpu().numpy(), wV)
    if q_heads:
        assert np.all(np.abs(read_o() - wo) <= tol)

    # Read back in every layout: byte * scale, one rounding; padding untouched.
    for back in ("token", "feature", "gaps", "strided"):
        bk, b_s, read_k = layout(np.full((tokens, f), 7.0, np.float32), back, rng)
        bv, _, read_v = layout(np.full((tokens, f), 8.0, np.float32), back, rng)
        assert lib.nnhip_kv8_read(pg, ptr(bk), *b_s, ptr(bv), *b_s, tokens, ptr(tseq) if with_seq else None, ptr(tpos), stream()) == 0
        want_k, want_v = np.full((tokens, f), 7.0, np.float32), np.full((tokens, f), 8.0, np.float32)
        for n in range(tokens):
            r, _ = ch.place(table, batch, page, pages, seq if with_seq else None, pos, 0, n)
            if r is not None:
                want_k[n] = (wK[r, :f].astype(np.float32).reshape(heads, dim) * wKs[r][:, None]).reshape(-1)
                want_v[n] = (wV[r, :f].astype(np.float32).reshape(heads, dim) * wVs[r][:, None]).reshape(-1)
        assert np.array_equal(read_k(), want_k, equal_nan=True) and np.array_equal(read_v(), want_v, equal_nan=True)
        if back == "gaps":
            assert np.all(bk.cpu().numpy().reshape(tokens, f + 3)[:, f:] == 77.0)
    only = dev(np.full((tokens, f), 7.0))
    assert lib.nnhip_kv8_read(pg, None, 0, 0, ptr(only), f, 1, tokens, ptr(tseq) if with_seq else None, ptr(tpos), stream()) == 0
    assert np.array_equal(only.cpu().numpy(), np.where(want_v == 8.0, 7.0, want_v), equal_nan=True)


# -- chunks of new tokens ----------------------------------------------------------
def cache_for(rng, lens, page, heads, dim, bits, holes=False, spare=2):
    """Caches and a table for sequences of these lengths; rows that none of them has hold NaN."""
    used = [-(-max(n, 0) // page) for n in lens]
    pages = sum(used) + spare
    width = max(max(used), 1) + 1
    table, at, order = np.full((len(lens), width), -1.0, np.float32), 0, rng.permutation(pages)
    for b, u in enumerate(used):
        table[b, :u] = order[at:at + u]
        at += u
    if holes:                  # absent positions, each way that an entry can be no page
        for b, u in enumerate(used):
            if u > 2:
                table[b, u // 2] = (np.nan, pages, -1)[b % 3]
    rows = pages * page
    read = np.zeros(rows, bool)
    for b, n in enumerate(lens):
        for j in range(n):
            r = ch.row_of(table, b, j, page, pages)
            if r is not None:
                read[r] = True
    if bits == 32:
        K, V = (rng.normal(size=(rows, heads, dim)).astype(np.float32) for _ in range(2))
        K[~read], V[~read] = np.nan, np.inf
        return dict(K=K, V=V, K64=K.astype(np.float64), V64=V.astype(np.float64)), table, pages
    x = dict()
    for n in "KV":
        x[n] = rng.integers(-127, 128, (rows, heads, dim)).astype(np.int8)
        x[n + "s"] = (rng.uniform(0.5, 2, (rows, heads)) * 2 / 127).astype(np.float32)
        x[n + "s"][~read] = np.nan
        x[n + "64"] = x[n].astype(np.float64) * x[n + "s"].astype(np.float64)[..., None]
    return x, table, pages


def run_chunk(x, c, table, q, start, most, lens, slopes, alpha, kind="token", stats=True, fill=9.0, at=None):
    """One call, twice: the same bits; O, m, l as arrays."""
    N, H, D = q.shape
    bits = 8 if "Ks" in x else 32
    lib, name = ch.library(), "nnhip_attn_chunk" + ("8" if bits == 8 else "")
    tq, sq, _ = layout(q.reshape(N, H * D), kind, None)
    to, so, read = layout(np.full((N, H * D), fill, np.float32), kind, None)
    flat = [x[n].reshape(len(x[n]), -1) for n in "KV"]
    if kind == "gaps":         # caches whose rows are longer than their heads, at any alignment
        flat = [np.concatenate([f, np.full((len(f), 3), 55, f.dtype)], 1) for f in flat]
        c = dict(c, row=flat[0].shape[1])
    tK, tV = (dev8(f) if bits == 8 else dev(f) for f in flat)
    if kind == "gaps":
        tK, tV = (torch.cat([t.reshape(-1)[:1], t.reshape(-1)])[1:] for t in (tK, tV))
    tKs, tVs = (dev(x[n + "s"]) if bits == 8 else None for n in "KV")
    tt, ts, tl = dev(table), dev(start), dev(lens)
    tsl = None if slopes is None else dev(slopes)
    m, l = torch.full((N, H), 4.0).cuda(), torch.full((N, H), 4.0).cuda()
    pg = pages_of(c, tK, tV, tt, tKs, tVs)
    need = getattr(lib, name + "_workspace_bytes")(pg, H, N, most)
    ws = torch.full((max(1, need // 4),), float("nan")).cuda()
    print(f"[chunk{bits}] tokens {N} most {most} batch {len(lens)} H {H} heads {c['heads']} dim {D} page {c['page']} {kind} ws {need}", flush=True)
    outs = []
    for _ in range(2):
        assert getattr(lib, name)(pg, ptr(tq), *sq, H, N, ptr(ts), most, ptr(tl), ptr(tsl), alpha, ptr(to), *so,
                                  ptr(m) if stats else None, ptr(l) if stats else None, ptr(ws) if need else None, need, stream()) == 0
        outs.append((read().reshape(N, H, D).copy(), m.cpu().numpy(), l.cpu().numpy()))
    assert all(np.array_equal(a, b, equal_nan=True) for a, b in zip(*outs))
    return outs[0]


def check_chunk(got, want, stats=True):
    """Where the 64-bit form is NaN (a NaN among the positions that a token sees) the result is, too."""
    O, m, l = got
    wO, wm, wl, tol, tol_m, has = want
    assert np.all(O[~has] == 9.0) and np.all(m[~has] == 4.0) and np.all(l[~has] == 4.0)
    assert np.array_equal(np.isnan(O[has]), np.isnan(wO[has]))
    bad = np.abs(O - wO)[has] > tol[has]
    assert not bad.any(), (np.argwhere(bad)[:5], (np.abs(O - wO)[has] / np.maximum(tol[has], 1e-35)).max())
    if stats:                  # l is a sum of weights, each off by twice what its score and m are, and by its sum's roundings (8192 positions at most)
        ok = has[:, None] & ~np.isnan(wm)
        assert np.all(np.abs(m - wm)[ok] <= tol_m[ok])
        assert np.all(np.abs(l - wl)[ok] <= wl[ok] * (4 * tol_m[ok] + (2 * 8192 + 8) * U))


CHUNK = [  # new tokens, past positions, q_heads, heads, dim, page, slopes, layout
    ([1], [0], 1, 1, 1, 1, False, "token"),
    ([1, 1, 1], [300, 0, 17], 12, 12, 64, 1, True, "feature"),
    ([5], [700], 12, 12, 64, 16, True, "feature"),
    ([3, 0, 1, 9], [40, 10, 0, 515], 8, 2, 128, 16, False, "token"),
    ([7, 16, 2], [33, 0, 100], 6, 3, 80, 24, True, "gaps"),
    ([40], [130], 6, 2, 96, 8, False, "feature"),
    ([17, 4], [700, 3], 4, 1, 128, 64, False, "strided"),
    ([12, 33], [90, 11], 3, 3, 30, 7, True, "token"),
    ([50], [0], 2, 2, 17, 1, False, "feature"),
    ([33, 1, 64], [50, 20, 0], 5, 1, 64, 16, False, "token"),
    ([130], [70], 2, 1, 20, 16, False, "token"),
    ([2], [4000], 1, 1, 128, 16, True, "token"),
    ([300], [31], 4, 2, 32, 16, True, "token"),
    ([129, 1, 257], [200, 999, 0], 4, 2, 128, 16, False, "feature"),
    ([70, 1, 1, 1], [600, 30, 1000, 5], 16, 4, 112, 16, True, "token"),
    ([1] * 70, list(range(70)), 2, 1, 64, 16, False, "token"),
    ([3] * 5 + [40] * 70, [9] * 75, 1, 1, 48, 16, False, "token"),
]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("new,past,q_heads,heads,dim,page,slopes,kind", CHUNK)
def test_chunk(new, past, q_heads, heads, dim, page, slopes, kind, bits):
    rng = np.random.default_rng(sum(new) * 31 + dim)
    lens = [n + p for n, p in zip(new, past)]
    x, table, pages = cache_for(rng, lens, page, heads, dim, bits, holes=len(new) % 2 == 0)
    start = np.concatenate([[0], np.cumsum(new)])
    q = rng.normal(size=(int(start[-1]), q_heads, dim)).astype(np.float32)
    sl = (2.0 ** -np.arange(1, q_heads + 1)).astype(np.float32) if slopes else None
    c = dict(pages=pages, page=page, heads=heads, dim=dim)
    alpha = np.float32(1.0 / math.sqrt(dim))
    most = max(new)
    got = run_chunk(x, c, table, q, start, most, lens, sl, alpha, kind)
    want = ch.attend(q, x["K64"], x["V64"], table, page, pages, heads, start, most, lens, float(alpha), sl)
    check_chunk(got, want)
    for kw in (dict(stats=False),):
        O, _, _ = run_chunk(x, c, table, q, start, most, lens, sl, alpha, kind, **kw)
        assert np.array_equal(O, got[0])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dim", [4, 8, 24, 28, 40, 44, 68, 72, 90, 100, 104, 116, 120, 127])
def test_head_widths(dim, bits):
    """Every width of the pieces that rows are read in, with up to 16, up to 32 and more rows of a key head."""
    rng = np.random.default_rng(dim)
    for new, past in (([4, 1], [90, 300]), ([7], [200]), ([7, 40, 1], [5, 60, 33])):
        lens, start = [n + p for n, p in zip(new, past)], np.concatenate([[0], np.cumsum(new)])
        x, table, pages = cache_for(rng, lens, 8, 2, dim, bits, holes=True)
        q = rng.normal(size=(int(start[-1]), 6, dim)).astype(np.float32)
        alpha = np.float32(1.0 / math.sqrt(dim))
        got = run_chunk(x, dict(pages=pages, page=8, heads=2, dim=dim), table, q, start, max(new), lens, None, alpha)
        check_chunk(got, ch.attend(q, x["K64"], x["V64"], table, 8, pages, 2, start, max(new), lens, float(alpha)))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("most,tokens", [(4, 40), (6, 70), (40, 200)])
def test_tokens_of_no_sequence(bits, most, tokens):
    """Tokens before the first sequence, behind the last, past `most`; sequences shorter than their chunk, of length 0, of
    NaN, longer than their table; starts that are negative, NaN or past the end: tokens of no sequence keep what they had,
    rows that see nothing get 0."""
    rng = np.random.default_rng(most)
    page, heads, dim, H = 8, 2, 64, 4
    n = [most, most + 3, 2, 0, most, 1, most]
    lens = [most + 50, 30, 1, 5, 0, 90, most // 2]
    x, table, pages = cache_for(rng, lens, page, heads, dim, bits)
    start = 3 + np.concatenate([[0], np.cumsum(n)]).astype(np.float32)
    q = rng.normal(size=(tokens, H, dim)).astype(np.float32)
    c = dict(pages=pages, page=page, heads=heads, dim=dim)
    ls = np.array(lens, np.float32)
    ls[5] = 1e9                # counts as the table's length; the pages behind the sequence's are absent
    variants = [(start, ls)]
    l2 = ls.copy()
    l2[0], l2[2] = np.nan, -7
    s2 = start.copy()
    s2[0], s2[-1] = -5, 1e9
    variants += [(start, l2), (s2, ls)]
    s3 = start.copy()
    s3[0] = np.nan
    variants += [(s3, ls)]
    for s, le in variants:
        got = run_chunk(x, c, table, q, s, most, le, None, 0.125)
        check_chunk(got, ch.attend(q, x["K64"], x["V64"], table, page, pages, heads, s, most, le, 0.125))


@pytest.mark.parametrize("new,past,per,dim", [(9, 20, 1, 64), (16, 64, 1, 128), (5, 0, 4, 30), (40, 100, 1, 64), (70, 10, 2, 128), (200, 33, 1, 96),
                                              (150, 500, 2, 64)])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_what_a_token_does_not_see(new, past, per, dim, value):
    """Keys and values that are not finite at a position change the tokens from there on, and none before. What the others
    get is what they get without, to rounding."""
    rng = np.random.default_rng(new + dim)
    page, heads = 16, 2
    lens, start = [new + past], [0, new]
    x, table, pages = cache_for(rng, lens, page, heads, dim, 32)
    c = dict(pages=pages, page=page, heads=heads, dim=dim)
    q = rng.normal(size=(new, heads * per, dim)).astype(np.float32)
    want = ch.attend(q, x["K64"], x["V64"], table, page, pages, heads, start, new, lens, 0.125)
    clean = run_chunk(x, c, table, q, start, new, lens, None, 0.125)
    check_chunk(clean, want)
    for at in sorted({1, new // 2, new - 1}):
        r = ch.row_of(table, 0, past + at, page, pages)
        for which in "VK":
            y = {n: a.copy() for n, a in x.items()}
            y[which][r, 0, dim // 2] = value
            O, m, l = run_chunk(y, c, table, q, start, new, lens, None, 0.125)
            assert np.all(np.abs(O[:at] - want[0][:at]) <= want[3][:at])
            assert np.all(np.abs(O[:, per:] - want[0][:, per:]) <= want[3][:, per:])
            if which == "V":
                assert not np.isfinite(O[at:, :per, dim // 2]).any()
                rest = np.arange(dim) != dim // 2
                assert np.all(np.abs(O[at:, :, rest] - want[0][at:, :, rest]) <= want[3][at:, :, rest])
            elif np.isnan(value):
                assert np.isnan(O[at:, :per]).all()
            else:              # +-inf q: a score of -inf is a position left out, one of +inf makes the row NaN
                up = np.sign(q[at:, :per, dim // 2]) * value > 0
                assert np.isnan(O[at:, :per][up]).all()
                y["K64"][r, 0, dim // 2] = value
                w2 = ch.attend(q, y["K64"], y["V64"], table, page, pages, heads, start, new, lens, 0.125)
                ok = np.abs(O[at:, :per] - w2[0][at:, :per])[~up] <= want[3][at:, :per][~up] * 4
                assert ok.all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("new,past,per,dim", [(9, 20, 1, 64), (5, 0, 4, 30), (20, 3, 1, 48), (40, 100, 1, 64), (70, 10, 2, 128), (200, 33, 1, 96)])
def test_large_values_that_a_token_does_not_see(new, past, per, dim, bits):
    """Finite keys and values of 1e30 among ordinary ones: the tokens in front of them are as exact as without."""
    rng = np.random.default_rng(new + dim)
    page, heads = 16, 2
    lens, start = [new + past], [0, new]
    x, table, pages = cache_for(rng, lens, page, heads, dim, bits)
    c = dict(pages=pages, page=page, heads=heads, dim=dim)
    q = rng.normal(size=(new, heads * per, dim)).astype(np.float32)
    want = ch.attend(q, x["K64"], x["V64"], table, page, pages, heads, start, new, lens, 0.125)
    for at in sorted({1, new // 2, new - 1}):
        r = ch.row_of(table, 0, past + at, page, pages)
        for which in "VK":
            y = {n: a.copy() for n, a in x.items()}
            if bits == 32:
                y[which][r] *= np.float32(1e30)
                y[which + "64"][r] = y[which][r]
            else:
                y[which + "s"][r] *= np.float32(1e30)
                y[which + "64"][r] = y[which][r].astype(np.float64) * y[which + "s"][r].astype(np.float64)[:, None]
            got = run_chunk(y, c, table, q, start, new, lens, None, 0.125)
            assert np.all(np.abs(got[0][:at] - want[0][:at]) <= want[3][:at])
            w2 = ch.attend(q, y["K64"], y["V64"], table, page, pages, heads, start, new, lens, 0.125)
            if bits == 8:      # bytes are held against the largest scale, not the largest product of one with its byte
                w2 = (*w2[:3], w2[3] + len(y["V64"]) * 2.0 ** -39 * 127 * np.abs(y["Vs"][np.isfinite(y["Vs"])]).max(), *w2[4:])
            check_chunk(got, w2, stats=False)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("new,lens", [([40], [0]), ([40], [float("nan")]), ([200], [-3]), ([200], [90]), ([50, 60, 3, 2], [0, 300, 0, 40]),
                                      ([50, 60, 70], [0, 0, 0]), ([40, 0, 33], [45, 20, 12])])
def test_lengths_below_the_chunks(new, lens, bits):
    """Sequences that are shorter than their chunk: tokens in front of the first position see nothing."""
    rng = np.random.default_rng(len(new))
    page, heads, dim = 16, 2, 64
    held = [int(n) if n > 0 else 0 for n in lens]
    x, table, pages = cache_for(rng, held, page, heads, dim, bits)
    start = np.concatenate([[0], np.cumsum(new)])
    q = rng.normal(size=(int(start[-1]), 2, dim)).astype(np.float32)
    got = run_chunk(x, dict(pages=pages, page=page, heads=heads, dim=dim), table, q, start, max(new), lens, None, 0.2)
    check_chunk(got, ch.attend(q, x["K64"], x["V64"], table, page, pages, heads, start, max(new), held, 0.2))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("new,past,per", [(5, 60, 2), (9, 40, 3), (70, 33, 1), (50, 9, 4)])
def test_factors_of_the_scores(new, past, per, bits):
    """alpha 0, negative and NaN; a query that is not finite, which changes its own row alone."""
    rng = np.random.default_rng(new)
    page, heads, dim = 16, 2, 48
    lens, start = [new + past], [0, new]
    x, table, pages = cache_for(rng, lens, page, heads, dim, bits)
    c = dict(pages=pages, page=page, heads=heads, dim=dim)
    q = rng.normal(size=(new, heads * per, dim)).astype(np.float32)
    sl = (2.0 ** -np.arange(1, heads * per + 1)).astype(np.float32)
    for alpha in (0.0, -0.3):
        for slopes in (None, sl):
            got = run_chunk(x, c, table, q, start, new, lens, slopes, np.float32(alpha))
            check_chunk(got, ch.attend(q, x["K64"], x["V64"], table, page, pages, heads, start, new, lens, float(np.float32(alpha)), slopes))
    assert np.isnan(run_chunk(x, c, table, q, start, new, lens, None, np.float32("nan"))[0]).all()
    clean = run_chunk(x, c, table, q, start, new, lens, None, np.float32(0.2))[0]
    want = ch.attend(q, x["K64"], x["V64"], table, page, pages, heads, start, new, lens, float(np.float32(0.2)))
    for value in (np.nan, np.inf):
        y = q.copy()
        y[2, 1, 3] = value
        O = run_chunk(x, c, table, y, start, new, lens, None, np.float32(0.2))[0]
        rest = np.ones(O.shape[:2], bool)
        rest[2, 1] = False
        assert np.all(np.abs(O - want[0])[rest] <= want[3][rest]) and np.all(np.abs(clean - want[0]) <= want[3])
        if bits == 8 or np.isnan(value):
            assert np.isnan(O[2, 1]).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_many_rows(bits):
    """Four million rows, long and single ones, the join's grid in two dimensions: some of them against the 64-bit form."""
    rng = np.random.default_rng(bits)
    page, heads, dim, qh, new, past = 64, 8, 4, 128, [8300, 1, 8300, 16600, 3], [5, 700, 0, 40, 90]
    lens, start = [n + p for n, p in zip(new, past)], np.concatenate([[0], np.cumsum(new)])
    x, table, pages = cache_for(rng, lens, page, heads, dim, bits)
    N = int(start[-1])
    assert N * qh > 1 << 22
    q = rng.normal(size=(N, qh, dim)).astype(np.float32)
    O, m, l = run_chunk(x, dict(pages=pages, page=page, heads=heads, dim=dim), table, q, start, max(new), lens, None, 0.5)
    for n in (0, 1, 8299, 8300, 8301, 12000, 16600, 16601, 30000, 33200, 33201, 33202, N - 1):
        b = int(np.searchsorted(start, n, side="right")) - 1
        seen = lens[b] - new[b] + n - int(start[b]) + 1
        for h in (0, 77, 127):   # the token alone, as the last of what it sees
            w = ch.attend(q[n:n + 1, h:h + 1], x["K64"][:, h // 16:h // 16 + 1], x["V64"][:, h // 16:h // 16 + 1], table[b:b + 1], page, pages, 1,
                          [0, 1], 1, [seen], 0.5)
            assert np.all(np.abs(O[n, h] - w[0][0, 0]) <= w[3][0, 0]) and abs(m[n, h] - w[1][0, 0]) <= w[4][0, 0]


@pytest.mark.parametrize("bits", [32, 8])
def test_few_rows_to_join(bits):
    """Prompts whose rows are whole, beside single tokens and a few whose ranges are joined."""
    rng = np.random.default_rng(bits)
    page, heads, dim, qh = 16, 8, 8, 64
    new, past = [900, 1, 0, 1000, 2, 4] + [1] * 14, [5, 700, 9, 40, 90, 0] + list(range(100, 800, 50))
    lens, start = [n + p for n, p in zip(new, past)], np.concatenate([[0], np.cumsum(new)])
    x, table, pages = cache_for(rng, lens, page, heads, dim, bits, holes=True)
    q = rng.normal(size=(int(start[-1]), qh, dim)).astype(np.float32)
    O, m, l = run_chunk(x, dict(pages=pages, page=page, heads=heads, dim=dim), table, q, start, max(new), lens, None, 0.5)
    for b, (lo, hi) in enumerate(zip(start[:-1], start[1:])):
        for n in range(lo, hi) if hi - lo < 5 else (lo, hi - 1):
            seen = lens[b] - new[b] + n - int(lo) + 1
            for h in range(0, qh, 7):
                w = ch.attend(q[n:n + 1, h:h + 1], x["K64"][:, h // 8:h // 8 + 1], x["V64"][:, h // 8:h // 8 + 1], table[b:b + 1], page, pages, 1,
                              [0, 1], 1, [seen], 0.5)
                assert np.all(np.abs(O[n, h] - w[0][0, 0]) <= w[3][0, 0]) and abs(m[n, h] - w[1][0, 0]) <= w[4][0, 0]
                assert abs(l[n, h] - w[2][0, 0]) <= w[2][0, 0] * (4 * w[4][0, 0] + (2 * 8192 + 8) * U)


@pytest.mark.parametrize("bits", [32, 8])
def test_table_of_many_positions(bits):
    """Tables that reach 2^24 positions: the keys' and values' parts are formed a sequence and key head at a time."""
    rng = np.random.default_rng(bits)
    page, heads, dim, new, past = 16, 2, 32, [40, 3, 100], [70, 50, 0]
    lens = [n + p for n, p in zip(new, past)]
    x, table, pages = cache_for(rng, lens, page, heads, dim, bits)
    wide = np.full((3, 1 << 20), -1, np.float32)
    wide[:, :table.shape[1]] = table
    start = np.concatenate([[0], np.cumsum(new)])
    q = rng.normal(size=(int(start[-1]), 4, dim)).astype(np.float32)
    got = run_chunk(x, dict(pages=pages, page=page, heads=heads, dim=dim), wide, q, start, 100, lens, None, 0.2)
    check_chunk(got, ch.attend(q, x["K64"], x["V64"], table, page, pages, heads, start, 100, lens, 0.2))


@pytest.mark.parametrize("new,past,per,dim", [(9, 20, 1, 64), (5, 0, 4, 30), (40, 100, 1, 64), (200, 33, 1, 96)])
def test_scales_that_are_not_finite(new, past, per, dim):
    """An 8-bit row that was not finite when it was stored (scale NaN) makes the tokens that see it NaN, and no other."""
    rng = np.random.default_rng(new + dim)
    page, heads = 16, 2
    lens, start = [new + past], [0, new]
    x, table, pages = cache_for(rng, lens, page, heads, dim, 8)
    c = dict(pages=pages, page=page, heads=heads, dim=dim)
    q = rng.normal(size=(new, heads * per, dim)).astype(np.float32)
    want = ch.attend(q, x["K64"], x["V64"], table, page, pages, heads, start, new, lens, 0.125)
    for at in sorted({1, new // 2, new - 1}):
        r = ch.row_of(table, 0, past + at, page, pages)
        for which in ("Vs", "Ks"):
            y = {n: a.copy() for n, a in x.items()}
            y[which][r, 0] = np.nan
            O, m, l = run_chunk(y, c, table, q, start, new, lens, None, 0.125)
            assert np.all(np.abs(O[:at] - want[0][:at]) <= want[3][:at]) and np.isnan(O[at:, :per]).all()
            assert np.all(np.abs(O[:, per:] - want[0][:, per:]) <= want[3][:, per:])


@pytest.mark.parametrize("new,past,dim", [(4, 100, 64), (40, 300, 64), (140, 300, 128)])
@pytest.mark.parametrize("k_size,v_size", [(1e-30, 1.0), (1e15, 1e-30), (1e30, 1e30), (1.0, 3e37), (1e-40, 1e-40)])
def test_sizes_of_values(new, past, dim, k_size, v_size):
    """Keys and values of any size that float32 holds, queries that bring the scores back to a few units; each row of the
    cache of a size of its own, within 2^-6 to 2^6."""
    rng = np.random.default_rng(new)
    page, heads = 16, 1
    lens, start = [new + past], [0, new]
    x, table, pages = cache_for(rng, lens, page, heads, dim, 32)
    rows = 2.0 ** rng.integers(-6, 1, (len(x["K"]), 1, 1))
    x["K"], x["V"] = (x["K"] * k_size * rows).astype(np.float32), (x["V"] * v_size * rows).astype(np.float32)
    x["K64"], x["V64"] = x["K"].astype(np.float64), x["V"].astype(np.float64)
    alpha = np.float32(0.125)
    q = (rng.normal(size=(new, 2, dim)) * min(1 / k_size, 1e37)).astype(np.float32)
    c = dict(pages=pages, page=page, heads=heads, dim=dim)
    got = run_chunk(x, c, table, q, start, new, lens, None, alpha)
    want = list(ch.attend(q, x["K64"], x["V64"], table, page, pages, heads, start, new, lens, float(alpha)))
    want[3] = want[3] + (new + past) * 2.0 ** -149   # denormal sums round to their own units
    check_chunk(got, want, stats=False)


@pytest.mark.parametrize("bits", [32, 8])
def test_scores_that_grow_and_fall(bits):
    """Scores that rise and fall by hundreds along the positions: the running maximum moves all the time."""
    rng = np.random.default_rng(3)
    page, heads, dim = 16, 1, 64
    for new, past in ((3, 900), (150, 700)):
        lens, start = [new + past], [0, new]
        x, table, pages = cache_for(rng, lens, page, heads, dim, bits)
        q = rng.normal(size=(new, 1, dim)).astype(np.float32)
        q[:, 0, 0] = 8.0
        for j in range(lens[0]):
            r = ch.row_of(table, 0, j, page, pages)
            big = 100 * np.sin(j / 40.0)
            if bits == 32:
                x["K"][r, 0, 0] = big
            else:
                x["K"][r, 0, 0] = np.sign(big) * 127
                x["Ks"][r, 0] = max(abs(big), 1) / 127
        x["K64"] = x["K"].astype(np.float64) * (1 if bits == 32 else x["Ks"].astype(np.float64)[..., None])
        c = dict(pages=pages, page=page, heads=heads, dim=dim)
        got = run_chunk(x, c, table, q, start, new, lens, None, 0.25)
        check_chunk(got, ch.attend(q, x["K64"], x["V64"], table, page, pages, heads, start, new, lens, 0.25), stats=False)


# -- verification --------------------------------------------------------------------
def run_verify(target, draft, fed, start, most, temperature, accept, pick, token_major, gap=0):
    N, V = target.shape
    lib = ch.library()

    def logits(x):
        if x is None:
            return None, V + gap if token_major else N + gap
        y = x if token_major else x.T
        y = np.concatenate([y, np.full((y.shape[0], gap), 1e30, np.float32)], 1)
        return dev(y), y.shape[1]

    (tt, t_ld), (td, d_ld) = logits(target), logits(draft)
    tf, ts = dev(fed), dev(start)
    ta, tp = (None if a is None else dev(a) for a in (accept, pick))
    B = len(start) - 1
    oa, ot = torch.full((B,), 7.5).cuda(), torch.full((B,), 7.5).cuda()
    need = lib.nnhip_draft_verify_workspace_bytes(N, B, most, V)
    ws = torch.full((need // 4 + 4,), float("nan")).cuda()
    print(f"[verify] tokens {N} batch {B} most {most} vocab {V} T {temperature} {'rows' if token_major else 'columns'} "
          f"{'no ' if draft is None else ''}draft", flush=True)
    for _ in range(2):
        assert lib.nnhip_draft_verify(ptr(tt), t_ld, ptr(td), d_ld, int(token_major), V, N, ptr(tf), ptr(ts), B, most, temperature,
                                      ptr(ta), ptr(tp), ptr(oa), ptr(ot), ptr(ws), need, stream()) == 0
        got = oa.cpu().numpy(), ot.cpu().numpy()
    return got


def drafted_batch(rng, counts, vocab, lead=0, tail=0):
    n = sum(counts) + lead + tail
    target = rng.normal(0, 2.5, (n, vocab)).astype(np.float32)
    draft = (target + rng.normal(0, 0.6, (n, vocab))).astype(np.float32)
    fed = np.zeros(n, np.float32)
    for i in range(n - 1):
        p = ch.softmax64(draft[i], 1.0)
        fed[i + 1] = min(int(np.searchsorted(np.cumsum(p), rng.uniform())), vocab - 1)
    start = (lead + np.concatenate([[0], np.cumsum(counts)])).astype(np.float32)
    return target, draft, fed, start, rng.uniform(size=n).astype(np.float32), rng.uniform(size=len(counts)).astype(np.float32)


VERIFY = [  # rows of each sequence, vocab
    ([1], 1), ([5], 1024), ([1, 1, 1], 50), ([4, 1, 0, 7, 2], 333), ([3] * 9, 32000), ([2, 9, 6], 100003), ([8] * 40, 700), ([33], 64),
    ([1], 512), ([2], 513), ([6] * 3, 4097),
]


@pytest.mark.parametrize("token_major", [True, False])
@pytest.mark.parametrize("temperature", [0.0, 1.0, 0.7])
@pytest.mark.parametrize("counts,vocab", VERIFY)
def test_verify(counts, vocab, temperature, token_major):
    rng = np.random.default_rng(sum(counts) * 7 + vocab)
    x = drafted_batch(rng, counts, vocab, lead=len(counts) % 2, tail=len(counts) % 3)
    target, draft, fed, start, accept, pick = x
    most = max(counts)
    for d in (draft, None):
        acc, tok, near = ch.verify(target, d, fed, start, most, temperature, accept, pick)
        assert near > 1e-12
        ga, gt = run_verify(target, d, fed, start, most, temperature, accept, pick, token_major, gap=3 if vocab == 333 else 0)
        assert np.array_equal(ga, acc) and np.array_equal(gt, tok)


@pytest.mark.parametrize("token_major", [True, False])
def test_verify_every_outcome(token_major):
    """All tokens stand, none does, each number of them; the numbers at their ends; special logits."""
    rng = np.random.default_rng(1)
    V, n = 700, 6
    target, draft, fed, start, accept, pick = drafted_batch(rng, [n] * 12, V)
    for b in range(12):
        lo = b * n
        accept[lo:lo + n] = 0.0
        if b < n - 1:
            accept[lo + b] = 1e30          # the b-th drafted token never stands
    pick[7], pick[8], pick[9], pick[10], pick[11] = 0.0, 1.0, np.nan, -3.0, 5.0
    draft[2 * n:3 * n] = target[2 * n:3 * n]           # p - q is 0 throughout: p
    target[3 * n + 3, 5], target[3 * n + 3, 9] = np.inf, np.inf
    target[4 * n + 4, :] = -np.inf
    target[0, ::2], target[0, 1] = np.nan, -np.inf
    target[11 * n:, V - 100:] = -np.inf                # the last token with a probability is not the last
    draft[1 * n + 1, :] = np.nan
    target[6 * n:7 * n] -= 3e38
    fed[5 * n + 2], fed[5 * n + 3] = V, np.nan
    acc, tok, near = ch.verify(target, draft, fed, start, n, 1.0, accept, pick)
    assert set(acc) >= {0, 1, 2, 3, 4, 5}
    ga, gt = run_verify(target, draft, fed, start, n, 1.0, accept, pick, token_major)
    assert np.array_equal(ga, acc) and np.array_equal(gt, tok)
    for d in (draft, None):
        for t in (0.0, 1e-30, 2.0):
            acc, tok, near = ch.verify(target, d, fed, start, n, t, accept, pick)
            ga, gt = run_verify(target, d, fed, start, n, t, accept, pick, token_major)
            assert np.array_equal(ga, acc) and np.array_equal(gt, tok)
    # fewer rows than a sequence has
    acc, tok, _ = ch.verify(target, draft, fed, start, 3, 1.0, accept, pick)
    ga, gt = run_verify(target, draft, fed, start, 3, 1.0, accept, pick, token_major)
    assert np.array_equal(ga, acc) and np.array_equal(gt, tok)


def test_verify_is_sampling():
    """With one row a sequence tokens are drawn from the softmax: over evenly spread numbers each token's share is its
    probability, to one number's share at either end."""
    V, n = 37, 4096
    rng = np.random.default_rng(0)
    z = rng.normal(0, 1.5, V).astype(np.float32)
    pick = ((np.arange(n) + 0.5) / n).astype(np.float32)
    start = np.arange(n + 1, dtype=np.float32)
    ga, gt = run_verify(np.tile(z, (n, 1)), None, np.zeros(n, np.float32), start, 1, 1.0, np.zeros(n, np.float32), pick, True)
    assert np.all(ga == 0)
    share = np.bincount(gt.astype(int), minlength=V) / n
    assert np.all(np.abs(share - ch.softmax64(z, 1.0)) <= 2.0 / n)


def test_verify_keeps_the_target_distribution():
    """Accepted tokens and replacements together are distributed as the target: summed over a grid of numbers, and drafted
    tokens in the draft's proportions, each token's share is its probability, to the grid's step."""
    V, reps, grid = 6, 600, 48
    rng = np.random.default_rng(2)
    zt, zd = rng.normal(0, 1, V).astype(np.float32), rng.normal(0, 1, V).astype(np.float32)
    q = ch.softmax64(zd, 1.0)
    token = np.minimum(np.searchsorted(np.cumsum(q), (np.arange(reps) + 0.5) / reps), V - 1)
    u, w = np.meshgrid((np.arange(grid) + 0.5) / grid, (np.arange(grid) + 0.5) / grid)
    seqs = grid * grid
    out = np.zeros(V)
    for x in range(V):
        n = 2 * seqs
        fed = np.zeros(n, np.float32)
        fed[1::2] = x
        accept = np.zeros(n, np.float32)
        accept[::2] = u.reshape(-1)
        ga, gt = run_verify(np.tile(zt, (n, 1)), np.tile(zd, (n, 1)), fed, np.arange(seqs + 1, dtype=np.float32) * 2, 2, 1.0, accept,
                            w.reshape(-1).astype(np.float32), True)
        first = np.where(ga == 1, x, gt)
        out += np.bincount(first.astype(int), minlength=V) / seqs * (token == x).mean()
    assert np.all(np.abs(out - ch.softmax64(zt, 1.0)) <= 2.0 / grid + 2.0 / reps)
