"""Paged caches and beam search's selection (include/nnhip_kernels.h: nnhip_kv_append, nnhip_attn_paged,
nnhip_beam_select, nnhip_kv_reorder) against plain 64-bit forms (paged_helpers.py).

Every buffer's untouched parts are checked as well: rows of the caches that no token names, the gaps of strided
outputs, padding. Rows that must not be read hold NaN.
"""
import math

import numpy as np
import pytest
import torch

import paged_helpers as ph

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def dev(a):
    return torch.as_tensor(np.ascontiguousarray(a, dtype=np.float32)).cuda()


def ptr(t):
    return None if t is None else t.data_ptr()


def stream():
    return torch.cuda.current_stream().cuda_stream


def cache(c, K, V, table):
    return ph.Pages(ptr(K), ptr(V), ptr(table), table.shape[0], table.shape[1], c["pages"], c["page"], c["heads"], c["dim"],
                    c.get("row", c["heads"] * c["dim"]))


def layout(x, kind, rng):
    """x (n, features) on the device: the buffer, its strides, and how to read it back."""
    n, f = x.shape
    if kind == "token":
        t = dev(x)
        return t, (f, 1), lambda: t.cpu().numpy()
    if kind == "feature":
        t = dev(x.T)
        return t, (1, n), lambda: t.cpu().numpy().T
    if kind == "gaps":         # rows 3 floats too long, one float off a 16-byte boundary
        buf = np.full(1 + n * (f + 3), 77.0, np.float32)
        view = buf[1:].reshape(n, f + 3)
        view[:, :f] = x
        t = dev(buf)
        return t[1:], (f + 3, 1), lambda: t.cpu().numpy()[1:].reshape(n, f + 3)[:, :f]
    t = dev(np.repeat(x.reshape(-1), 2))   # "strided": every other float
    return t, (2 * f, 2), lambda: t.cpu().numpy()[::2].reshape(n, f)


# -- append --------------------------------------------------------------------
APPEND = [  # tokens, batch, q_heads, heads, dim, rope, page, layout, seq
    (1, 1, 1, 1, 1, 0, 1, "token", True),
    (4, 4, 12, 12, 64, 64, 1, "feature", False),
    (3, 2, 2, 1, 2, 2, 3, "token", True),
    (33, 5, 8, 2, 128, 128, 16, "token", True),
    (70, 3, 6, 6, 80, 40, 64, "feature", True),
    (65, 7, 3, 3, 30, 28, 24, "gaps", True),
    (50, 2, 4, 2, 17, 6, 8, "strided", True),
    (40, 3, 2, 2, 256, 256, 16, "token", True),
    (129, 1, 4, 4, 36, 36, 7, "feature", True),
    (9, 9, 0, 4, 64, 64, 16, "feature", False),
]


@pytest.mark.parametrize("tokens,batch,q_heads,heads,dim,rope,page,kind,with_seq", APPEND)
def test_append(tokens, batch, q_heads, heads, dim, rope, page, kind, with_seq):
    rng = np.random.default_rng(tokens * 131 + dim)
    per = -(-tokens // batch) + 5
    width = -(-per // page) + 1
    pages = batch * width + 2
    c = dict(pages=pages, page=page, heads=heads, dim=dim, row=heads * dim + (5 if kind == "gaps" else 0))
    table = rng.permutation(pages)[:batch * width].reshape(batch, width).astype(np.float32)
    if with_seq:
        order = rng.permutation(batch * per)[:tokens]
        seq, pos = order // per, (order % per).astype(np.float32)
    else:
        seq, pos = np.arange(tokens), rng.integers(0, per, tokens).astype(np.float32)
    rope_rows = per - 2
    pos_b = pos.copy()
    if tokens >= 30:           # padding: no position, no sequence, no page, no row of the rotation
        pos_b[3], pos_b[5], pos_b[7], pos_b[11] = -1, np.nan, width * page, 2.0 ** 30
        table[0, 0], table[batch - 1, width - 1] = -1, np.nan
        table[batch // 2, 0] = pages
    seq_f = seq.astype(np.float32)
    if tokens >= 30:
        seq_f[13], seq_f[17], seq_f[19] = -1, batch, np.nan
    row = c["row"]
    k, v = (rng.normal(size=(tokens, heads * dim)).astype(np.float32) for _ in range(2))
    q = rng.normal(size=(tokens, max(1, q_heads) * dim)).astype(np.float32)
    ang = rng.uniform(-3, 3, (rope_rows, max(1, rope // 2)))
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    K0, V0 = (rng.normal(size=(pages * page, row)).astype(np.float32) for _ in range(2))
    (tk, sk, _), (tv, sv, _), (tq, sq, _) = (layout(x, kind, rng) for x in (k, v, q))
    out0 = np.full_like(q, 5.0)
    to, so, read_o = layout(out0, "feature" if kind == "token" else kind, rng)
    K, V, tt, tc, tsn = dev(K0), dev(V0), dev(table), dev(cos), dev(sin)
    tseq, tpos = dev(seq_f), dev(pos_b)
    print(f"[append] {tokens} tokens heads {heads} dim {dim} rope {rope} page {page} {kind}", flush=True)
    rc = ph.library().nnhip_kv_append(
        cache(c, K, V, tt), ptr(tk), *sk, ptr(tv), *sv, ptr(tq) if q_heads else None, *sq, ptr(to) if q_heads else None,
        *so, q_heads, tokens, ptr(tseq) if with_seq else None, ptr(tpos), ptr(tc) if rope else None,
        ptr(tsn) if rope else None, rope_rows if rope else 0, rope, stream())
    assert rc == 0
    wK, wV, wo = K0.astype(np.float64), V0.astype(np.float64), out0.astype(np.float64)
    tol_k, tol_o = np.zeros_like(wK), np.zeros_like(wo)
    h = rope // 2

    def turned(x, p):
        """Rotated value and its bound: two products and an addition, each rounded (2^-23 of the terms' sizes)."""
        x = x.astype(np.float64).reshape(-1, dim)
        y, size = x.copy(), np.zeros_like(x)
        if h:
            co, si = cos[p].astype(np.float64), sin[p].astype(np.float64)
            y[:, :h] = x[:, :h] * co - x[:, h:2 * h] * si
            y[:, h:2 * h] = x[:, h:2 * h] * co + x[:, :h] * si
            size[:, :h] = size[:, h:2 * h] = np.abs(x[:, :h] * co) + np.abs(x[:, h:2 * h] * si)
            size[:, h:2 * h] = np.abs(x[:, h:2 * h] * co) + np.abs(x[:, :h] * si)
        return y.reshape(-1), 2 * U * size.reshape(-1)

    for n in range(tokens):
        b = ph.index_of(seq_f[n], batch)
        p = ph.index_of(pos_b[n], 1 << 24)
        if b is None or p is None or (rope and p >= rope_rows):
            continue
        r = ph.row_of(table, b, p, page, pages)
        if r is None:
            continue
        wK[r, :heads * dim], tol_k[r, :heads * dim] = turned(k[n], p)
        wV[r, :heads * dim] = v[n]
        if q_heads:
            wo[n], tol_o[n] = turned(q[n], p)
    assert np.all(np.abs(K.cpu().numpy() - wK) <= tol_k)
    assert np.array_equal(V.cpu().numpy(), wV.astype(np.float32))
    if q_heads:
        assert np.all(np.abs(read_o() - wo) <= tol_o)


def test_append_in_place():
    """q_out may be q itself."""
    rng = np.random.default_rng(5)
    n, h, d = 37, 4, 32
    c = dict(pages=40, page=1, heads=h, dim=d)
    q, k, v = (dev(rng.normal(size=(n, h * d))) for _ in range(3))
    K, V, table = torch.zeros(40, h * d).cuda(), torch.zeros(40, h * d).cuda(), dev(np.arange(40)[None, :])
    cos, sin = dev(np.cos(rng.uniform(0, 6, (40, d // 2)))), dev(np.sin(rng.uniform(0, 6, (40, d // 2))))
    seq, pos, out = torch.zeros(n).cuda(), dev(np.arange(n)), torch.zeros_like(q)
    lib = ph.library()
    for o in (out, q):
        assert lib.nnhip_kv_append(cache(c, K, V, table), ptr(k), h * d, 1, ptr(v), h * d, 1, ptr(q), h * d, 1, ptr(o), h * d,
                                   1, h, n, ptr(seq), ptr(pos), ptr(cos), ptr(sin), 40, d, stream()) == 0
    assert torch.equal(out, q)


# -- attention -------------------------------------------------------------------
def batch_of(rng, groups, beams, page, prefix, lens, share, extra=1):
    """Page tables of groups whose sequences share the whole pages of their first `prefix` positions."""
    B = groups * beams
    width = -(-max(max(lens), 1) // page) + extra
    table = np.full((B, width), -1.0, np.float32)
    used = 0
    for g in range(groups):
        full = prefix[g] // page if share else 0
        table[g * beams:(g + 1) * beams, :full] = np.arange(used, used + full)
        used += full
        for b in range(g * beams, (g + 1) * beams):
            need = max(0, -(-lens[b] // page) - full)
            table[b, full:full + need] = np.arange(used, used + need)
            used += need
    pages = used + 2
    perm = rng.permutation(pages)
    live = table >= 0
    table[live] = perm[table[live].astype(int)]
    return table, pages


def run_attend(c, q, K, V, table, lens, shared, group, slopes, alpha, kind="token", stats=True):
    B, H, D = q.shape
    lib = ph.library()
    tq, sq, _ = layout(q.reshape(B, H * D), kind, None)
    to, so, read = layout(np.full((B, H * D), 9.0, np.float32), kind, None)
    tK, tV, tt, tl = dev(K.reshape(len(K), -1)), dev(V.reshape(len(V), -1)), dev(table), dev(lens)
    if c.get("offset"):        # caches one float off a 16-byte boundary
        tK, tV = (torch.cat([torch.zeros(1).cuda(), t.reshape(-1)])[1:] for t in (tK, tV))
    ts = None if shared is None else dev(shared)
    tsl = None if slopes is None else dev(slopes)
    m, l = torch.full((B, H), 4.0).cuda(), torch.full((B, H), 4.0).cuda()
    pg = cache(c, tK, tV, tt)
    need = lib.nnhip_attn_paged_workspace_bytes(pg, H, group)
    ws = torch.full((max(1, need // 4),), float("nan")).cuda()
    print(f"[attend] B {B} group {group} H {H} heads {c['heads']} dim {D} page {c['page']} width {table.shape[1]} {kind} "
          f"ws {need}", flush=True)
    outs = []
    for _ in range(2):
        rc = lib.nnhip_attn_paged(pg, ptr(tq), *sq, H, ptr(tl), ptr(ts), group, ptr(tsl), alpha, ptr(to), *so,
                                  ptr(m) if stats else None, ptr(l) if stats else None, ptr(ws) if need else None, need,
                                  stream())
        assert rc == 0
        outs.append((read().reshape(B, H, D).copy(), m.cpu().numpy(), l.cpu().numpy()))
    assert all(np.array_equal(x, y, equal_nan=True) for x, y in zip(*outs))
    return outs[0]


def poison(K, V, table, lens, page, pages):
    """NaN and infinities in every row that no sequence reads."""
    read = {ph.row_of(table, b, j, page, pages) for b in range(len(lens))
            for j in range(ph.length_of(lens[b], table.shape[1] * page))}
    for r in range(len(K)):
        if r not in read:
            K[r], V[r] = (np.nan, np.inf) if r % 2 else (-np.inf, np.nan)


ATTEND = [  # groups, beams, q_heads, heads, dim, page, prefix, longest own part, share, slopes, layout
    (1, 1, 1, 1, 1, 1, 1, 1, False, False, "token"),
    (1, 4, 12, 12, 64, 1, 300, 21, True, True, "feature"),
    (2, 3, 4, 4, 32, 16, 100, 40, True, False, "token"),
    (1, 7, 8, 2, 128, 16, 515, 33, True, True, "token"),
    (3, 1, 6, 3, 80, 24, 200, 9, False, True, "gaps"),
    (1, 40, 6, 2, 96, 8, 130, 70, True, False, "feature"),
    (2, 20, 4, 1, 128, 64, 700, 3, True, False, "strided"),
    (1, 5, 3, 3, 30, 7, 90, 11, True, True, "token"),
    (1, 3, 2, 2, 17, 1, 64, 2, True, False, "feature"),
    (4, 2, 40, 1, 64, 16, 50, 20, True, False, "token"),
    (1, 70, 2, 1, 20, 16, 33, 18, False, False, "token"),
    (1, 2, 1, 1, 128, 16, 4000, 100, True, False, "token"),
    (5, 1, 2, 2, 64, 16, 1, 1, True, False, "token"),
]


@pytest.mark.parametrize("groups,beams,q_heads,heads,dim,page,prefix,own,share,slopes,kind", ATTEND)
def test_attend(groups, beams, q_heads, heads, dim, page, prefix, own, share, slopes, kind):
    rng = np.random.default_rng(groups * 1009 + beams * 31 + dim)
    pre = [prefix] + [int(rng.integers(1, prefix + 1)) for _ in range(groups - 1)]
    lens = [pre[b // beams] + int(rng.integers(0, own + 1)) for b in range(groups * beams)]
    lens[0] = prefix + own
    table, pages = batch_of(rng, groups, beams, page, pre, lens, share)
    K, V = (rng.normal(size=(pages * page, heads, dim)).astype(np.float32) for _ in range(2))
    poison(K, V, table, lens, page, pages)
    q = rng.normal(size=(groups * beams, q_heads, dim)).astype(np.float32)
    sl = (2.0 ** -np.arange(1, q_heads + 1)).astype(np.float32) if slopes else None
    shared = [n // page * page for n in pre] if share else None
    c = dict(pages=pages, page=page, heads=heads, dim=dim, offset=kind == "gaps")
    alpha = 1.0 / math.sqrt(dim)
    O, m, l = run_attend(c, q, K, V, table, lens, shared, beams, sl, alpha, kind)
    wO, wm, wl, tol = ph.attend(q, K, V, table, page, pages, heads, lens, alpha, sl)
    assert np.all(np.abs(O - wO) <= tol + 1e-30)
    # m is one score, l a sum of weights that are each off by what scores and m are
    s_tol = (dim + 8) * U * np.abs(q).sum(axis=2) * np.abs(K[np.isfinite(K)]).max() * alpha + 8 * U * np.abs(wm)
    assert np.all(np.abs(m - wm) <= s_tol)
    assert np.all(np.abs(l - wl) <= wl * (4 * s_tol + 2 * max(lens) * U))


@pytest.mark.parametrize("kind", ["token", "gaps", "feature", "strided"])
@pytest.mark.parametrize("heads,per,beams,dim", [(2, 2, 3, 64), (1, 3, 2, 20), (2, 20, 2, 128), (1, 1, 1, 80), (2, 1, 40, 32)])
def test_attend_query_layouts(heads, per, beams, dim, kind):
    """Queries of any alignment beside aligned caches."""
    rng = np.random.default_rng(dim + beams)
    prefix, page = 70, 16
    lens = [prefix + int(n) for n in rng.integers(0, 20, beams)]
    table, pages = batch_of(rng, 1, beams, page, [prefix], lens, True)
    K, V = (rng.normal(size=(pages * page, heads, dim)).astype(np.float32) for _ in range(2))
    q = rng.normal(size=(beams, heads * per, dim)).astype(np.float32)
    c = dict(pages=pages, page=page, heads=heads, dim=dim)
    O, _, _ = run_attend(c, q, K, V, table, lens, [prefix // page * page], beams, None, 0.2, kind)
    wO, _, _, tol = ph.attend(q, K, V, table, page, pages, heads, lens, np.float32(0.2))
    assert np.all(np.abs(O - wO) <= tol + 1e-30)


# Many rows to a position (more than 32): the products are formed from bf16 parts, and again in float32 where these
# do not hold the values.
def many_rows(rng, beams, per, dim, prefix, own, page=16):
    lens = [prefix + int(rng.integers(1, own + 1)) for _ in range(beams)]
    lens[0] = prefix + own
    table, pages = batch_of(rng, 1, beams, page, [prefix], lens, True)
    K, V = (rng.normal(size=(pages * page, 1, dim)).astype(np.float32) for _ in range(2))
    q = rng.normal(size=(beams, per, dim)).astype(np.float32)
    return dict(pages=pages, page=page, heads=1, dim=dim), q, K, V, table, lens, [prefix // page * page]


def check_many(c, q, K, V, table, lens, shared, alpha, slopes=None):
    beams = q.shape[0]
    O, m, l = run_attend(c, q, K, V, table, lens, shared, beams, slopes, alpha)
    wO, wm, wl, tol = ph.attend(q, K, V, table, c["page"], c["pages"], 1, lens, alpha, slopes)
    assert np.array_equal(np.isfinite(O), np.isfinite(wO))
    ok = np.isfinite(wO)
    assert np.all(np.abs(O[ok] - wO[ok]) <= tol[ok])
    return O


@pytest.mark.parametrize("beams,per,dim,prefix,own", [(9, 4, 32, 130, 20), (33, 1, 64, 400, 9), (40, 3, 96, 700, 5),
                                                     (16, 4, 128, 1500, 40), (70, 2, 128, 333, 3), (40, 1, 80, 200, 7),
                                                     (20, 2, 48, 300, 4), (3, 20, 128, 200, 50), (2, 17, 64, 129, 2)])
@pytest.mark.parametrize("slopes", [False, True])
def test_attend_many_rows(beams, per, dim, prefix, own, slopes):
    rng = np.random.default_rng(beams * 100 + dim)
    c, q, K, V, table, lens, shared = many_rows(rng, beams, per, dim, prefix, own)
    poison(K, V, table, lens, c["page"], c["pages"])
    lens[1] = shared[0] - 3            # one reads its own table, one nothing
    if beams > 2:
        lens[2] = 0
    sl = (2.0 ** -np.arange(3, per + 3)).astype(np.float32) if slopes else None
    check_many(c, q, K, V, table, lens, shared, 1 / math.sqrt(dim), sl)


@pytest.mark.parametrize("what", ["keys 2^104", "keys 2^127", "queries 2^110", "values 2^104", "values 2^126", "scores 2^90",
                                  "scores -2^90", "tiny", "tiny values", "alpha 2^-70", "key -inf", "key inf", "key nan",
                                  "value inf", "value nan", "query nan", "wide values"])
def test_attend_many_rows_range(what):
    rng = np.random.default_rng(len(what))
    c, q, K, V, table, lens, shared = many_rows(rng, 12, 4, 64, 300, 6)
    alpha = 0.125
    at = ph.row_of(table, 0, 77, c["page"], c["pages"])
    if what.startswith("keys"):        # one dim of the keys, which the queries weigh as little
        e = int(what.split("^")[1])
        K[:, 0, 5] *= np.float32(2.0 ** (e - 2))
        q[:, :, 5] *= np.float32(2.0 ** -(e - 1))
    elif what == "queries 2^110":
        q[:, :, 5] *= np.float32(2.0 ** 110)
        K[:, 0, 5] *= np.float32(2.0 ** -111)
    elif what.startswith("values 2"):
        V *= np.float32(2.0 ** (int(what.split("^")[1]) - 3))
    elif what == "scores 2^90":
        q *= np.float32(2.0 ** 45)
        K *= np.float32(2.0 ** 45)
    elif what == "scores -2^90":       # every score far below any sum that the parts hold
        q, K = -np.abs(q) * np.float32(2.0 ** 45), np.abs(K) * np.float32(2.0 ** 45)
    elif what == "tiny":
        q *= np.float32(2.0 ** -60)
        K *= np.float32(2.0 ** -66)
        alpha = 2.0 ** 123
    elif what == "tiny values":
        V *= np.float32(2.0 ** -120)
    elif what == "alpha 2^-70":
        q *= np.float32(2.0 ** 34)
        K *= np.float32(2.0 ** 34)
        alpha = 2.0 ** -70
    elif what == "key -inf":
        K[at, 0, 3] = -np.inf
        q[:, :, 3] = np.abs(q[:, :, 3]) + 0.5
    elif what == "key inf":
        K[at, 0, 3] = np.inf
        q[:, :, 3] = np.abs(q[:, :, 3]) + 0.5
    elif what == "key nan":
        K[at, 0, 3] = np.nan
    elif what == "value inf":
        V[at, 0, 3] = np.inf
    elif what == "value nan":
        V[at, 0, 3] = np.nan
    elif what == "query nan":
        q[4, 2, 1] = np.nan
    elif what == "wide values":
        V *= (2.0 ** rng.integers(-60, 60, V.shape)).astype(np.float32)
    O = check_many(c, q, K, V, table, lens, shared, alpha)
    if what == "query nan":
        assert np.isnan(O[4, 2]).all() and np.isfinite(np.delete(O.reshape(48, 64), 18, 0)).all()


@pytest.mark.parametrize("slopes,falls,size", [(0, False, 0), (0, False, 60), (0, False, 600), (0, False, 900), (0, False, 1000),
                                               (0, False, 1100), (0, False, 1300), (0, True, 60), (0, True, 600),
                                               (0.25, False, 0), (3.0, False, 0), (3.0, True, 60), (3.0, True, 20000),
                                               (-2.0, False, 0), (0.01, False, 300)])
def test_attend_many_rows_far_scores(slopes, falls, size):
    """Several tiles a wave, over which the scores grow or fall along the positions, by themselves or by the slope."""
    rng = np.random.default_rng(int(size) + 7)
    heads, per, beams, dim, n, page = 16, 4, 10, 32, 8000, 16
    lens = [n + int(x) for x in rng.integers(1, 9, beams)]
    table, pages = batch_of(rng, 1, beams, page, [n], lens, True)
    K, V = (rng.normal(size=(pages * page, heads, dim)).astype(np.float32) for _ in range(2))
    q = rng.normal(size=(beams, heads * per, dim)).astype(np.float32) * np.float32(0.25)
    ramp = np.linspace(size, 0, n) if falls else np.linspace(0, size, n)
    for j in range(n):
        K[ph.row_of(table, 0, j, page, pages), :, 0] = np.float32(ramp[j])
    q[:, :, 0] = 1.0
    sl = (slopes * np.linspace(0.5, 1, heads * per)).astype(np.float32) if slopes else None
    c = dict(pages=pages, page=page, heads=heads, dim=dim)
    O, m, l = run_attend(c, q, K, V, table, lens, [n], beams, sl, 1.0)
    wO, wm, wl, tol = ph.attend(q, K, V, table, page, pages, heads, lens, 1.0, sl)
    assert np.all(np.abs(O - wO) <= tol)
    # as in test_attend; the slope's product with up to 8000 is rounded too
    s_tol = (dim + 8) * U * np.abs(q).sum(axis=2) * np.abs(K).max() + 8 * U * np.abs(wm)
    if slopes:
        s_tol = s_tol + 2 * U * np.abs(sl)[None, :] * n
    assert np.all(np.abs(m - wm) <= s_tol)
    assert np.all(np.abs(l - wl) <= wl * (4 * s_tol + 2 * max(lens) * U))


def test_attend_lengths_and_pages():
    """Lengths of zero, one, below the shared prefix, NaN, negative and beyond the table; pages that do not exist in
    the prefix, in a sequence's own part and at its end; infinities in rows that another sequence reads."""
    rng = np.random.default_rng(3)
    beams, page, heads, dim = 10, 8, 2, 64
    prefix = [40]
    lens = [90, 0, 1, 39, 40, 41, 90, 77, 90, 64]
    table, pages = batch_of(rng, 1, beams, page, prefix, lens, True)
    K, V = (rng.normal(size=(pages * page, heads, dim)).astype(np.float32) for _ in range(2))
    lens_f = np.array(lens, np.float32)
    lens_f[6], lens_f[7], lens_f[8] = np.nan, -5.0, 1e9
    table[:, 2] = -1.0                 # a hole in the prefix
    table[5, 5], table[8, 9], table[9, 7] = pages, np.nan, -7
    poison(K, V, table, lens_f, page, pages)
    # Position 39 belongs to the sequences that are at least 40 long: the one of 39 must not see its infinities.
    r = ph.row_of(table, 0, 39, page, pages)
    K[r, 1], V[r, 1] = np.inf, np.inf
    q = rng.normal(size=(beams, heads, dim)).astype(np.float32)
    c = dict(pages=pages, page=page, heads=heads, dim=dim)
    for shared in ([40.0], [37.0], [0.0], [np.nan], [-3.0], None, [41.0]):
        if shared == [41.0]:           # more than the tables have in common for the shorter ones: all read their own
            lens_f[[0, 4, 5, 8, 9]] = [40, 40, 40, 40, 40]
        O, m, l = run_attend(c, q, K, V, table, lens_f, shared, beams, None, 0.125)
        wO, wm, wl, tol = ph.attend(q, K, V, table, page, pages, heads, lens_f, 0.125)
        assert np.array_equal(np.isnan(O), np.isnan(wO))
        ok = ~np.isnan(wO)
        assert np.all(np.abs(O - wO)[ok] <= tol[ok] + 1e-30)
        for b in (1, 6, 7):
            assert np.all(O[b] == 0) and np.all(l[b] == 0) and np.all(m[b] == np.float32(-3.40282347e38))


def test_attend_scores_of_minus_infinity():
    """Every score -inf gives 0, as no position does; one NaN key gives NaN to its heads alone."""
    rng = np.random.default_rng(4)
    n, dim = 50, 32
    K, V = (rng.normal(size=(64, 2, dim)).astype(np.float32) for _ in range(2))
    K[:, 0, 3] = -np.inf
    K[17, 1, 0] = np.nan
    q = np.abs(rng.normal(size=(2, 4, dim))).astype(np.float32) + 0.1
    table = np.arange(4, dtype=np.float32)[None, :].repeat(2, 0)
    c = dict(pages=4, page=16, heads=2, dim=dim)
    for shared in (None, [48.0]):
        O, m, l = run_attend(c, q, K, V, table, [n, 17], shared, 2, None, 1.0)
        assert np.all(O[:, :2] == 0) and np.all(l[:, :2] == 0)
        assert np.all(np.isnan(O[0, 2:])) and not np.isnan(O[1]).any()


@pytest.mark.parametrize("at,n", [(0, 1), (0, 300), (16, 17), (70, 71), (299, 300), (150, 300)])
@pytest.mark.parametrize("shared", [None, 288])
def test_attend_one_nan(at, n, shared):
    """One NaN key, alone in its tile, its wave or its range or not, makes the sequences that see it NaN, and no other."""
    rng = np.random.default_rng(at + n)
    K, V = (rng.normal(size=(304, 1, 64)).astype(np.float32) for _ in range(2))
    K[at] = np.nan
    q = rng.normal(size=(2, 2, 64)).astype(np.float32)
    table = np.arange(19, dtype=np.float32)[None, :].repeat(2, 0)
    c = dict(pages=19, page=16, heads=1, dim=64)
    O, m, l = run_attend(c, q, K, V, table, [n, at], None if shared is None else [shared], 2, None, 1.0)
    assert np.isnan(O[0]).all() and np.isnan(l[0]).all() and not np.isnan(O[1]).any()


def test_attend_large_scores():
    """Scores around 1e4 in both directions: exact weights of 0 and 1, no overflow."""
    rng = np.random.default_rng(8)
    n, dim = 300, 64
    K, V = (rng.normal(size=(304, 1, dim)).astype(np.float32) for _ in range(2))
    q = (rng.normal(size=(3, 1, dim)) * 1000).astype(np.float32)
    table = np.arange(19, dtype=np.float32)[None, :].repeat(3, 0)
    c = dict(pages=19, page=16, heads=1, dim=dim)
    O, m, l = run_attend(c, q, K, V, table, [n] * 3, [288.0], 3, None, 1.0)
    s = q[:, 0].astype(np.float64) @ K[:n, 0].astype(np.float64).T
    top2 = np.sort(s, axis=1)[:, -2:]
    assert (top2[:, 1] - top2[:, 0]).min() > 30      # one weight is 1 to float32
    assert np.all(np.abs(O[:, 0] - V[s.argmax(axis=1), 0]) <= 1e-6)


def test_attend_far_rows():
    """Rows beyond 2^31 floats and 2^33 bytes of the caches, appended and read back."""
    heads, dim, page = 8, 128, 256
    pages = 9001
    rows, row = pages * page, heads * dim
    K, V = torch.empty(rows, row, device="cuda"), torch.empty(rows, row, device="cuda")
    assert K.numel() > 2 ** 31
    rng = np.random.default_rng(9)
    B, n = 3, 300
    table_h = np.array([[pages - 1, pages - 3], [pages - 1, pages - 5], [pages - 1, 8400]], np.float32)
    table = dev(table_h)
    lens = [n, n - 20, 256 + 1]
    k, v = (rng.normal(size=(B * n, row)).astype(np.float32) for _ in range(2))
    seq, pos = np.repeat(np.arange(B), n), np.tile(np.arange(n), B).astype(np.float32)
    pos[(seq > 0) & (pos < page)] = -1       # the shared page is written once
    pos[pos >= np.array(lens)[seq]] = -1
    tk, tv, ts, tp = dev(k), dev(v), dev(seq), dev(pos)
    c = dict(pages=pages, page=page, heads=heads, dim=dim)
    pg = cache(c, K, V, table)
    lib = ph.library()
    assert lib.nnhip_kv_append(pg, ptr(tk), row, 1, ptr(tv), row, 1, None, 0, 0, None, 0, 0, 0, B * n, ptr(ts), ptr(tp), None,
                               None, 0, 0, stream()) == 0
    q = rng.normal(size=(B, heads, dim)).astype(np.float32)
    tq, out, tl, tsh = dev(q), torch.zeros(B, row).cuda(), dev(lens), dev([page])
    need = lib.nnhip_attn_paged_workspace_bytes(pg, heads, B)
    ws = torch.empty(need // 4, device="cuda")
    assert lib.nnhip_attn_paged(pg, ptr(tq), row, 1, heads, ptr(tl), ptr(tsh), B, None, 0.1, ptr(out), row, 1, None, None,
                                ptr(ws), need, stream()) == 0
    kk, vv = (x.reshape(B, n, heads, dim) for x in (k, v))
    got = out.cpu().numpy().reshape(B, heads, dim)
    for b in range(B):
        kb = np.concatenate([kk[0, :page], kk[b, page:lens[b]]])
        vb = np.concatenate([vv[0, :page], vv[b, page:lens[b]]])
        t1 = np.arange(lens[b], dtype=np.float32)[None, :]
        wO, _, _, tol = ph.attend(q[b:b + 1], kb, vb, t1, 1, lens[b], heads, [lens[b]], np.float32(0.1))
        assert np.all(np.abs(got[b] - wO[0]) <= tol[0])
    # a page copied far out
    parent, fresh, tl2 = dev([0.0, 1.0, 2.0]), dev([8990.0, 8991.0, 8992.0]), dev(lens)
    tout, lout = torch.zeros(3, 2).cuda(), torch.zeros(3).cuda()
    assert lib.nnhip_kv_reorder((ph.Pages * 1)(pg), 1, ptr(parent), ptr(tl2), ptr(fresh), 3, ptr(tout), ptr(lout),
                                stream()) == 0
    for b in range(B):
        src, dst, tail = int(table_h[b, 1]) * page, (8990 + b) * page, lens[b] - page
        assert torch.equal(K[dst:dst + tail], K[src:src + tail]) and torch.equal(V[dst:dst + tail], V[src:src + tail])


# -- selection -------------------------------------------------------------------
SELECT = [  # groups, beams, vocab, take, beam_major, ended
    (1, 1, 1, 1, True, 0), (1, 1, 1, 1, False, 0), (1, 2, 3, 6, True, 1), (1, 2, 3, 6, False, 1),
    (1, 4, 1024, 8, False, 1), (2, 3, 1000, 6, False, 0), (1, 16, 5003, 32, False, 2), (7, 5, 777, 10, True, 1),
    (3, 8, 20011, 16, True, 0), (1, 1, 257, 256, True, 0), (1, 1, 65, 64, False, 0), (2, 33, 130, 40, False, 7),
    (1, 1024, 64, 256, False, 0), (1, 300, 100, 256, True, 20), (40, 2, 129, 5, False, 0), (1, 8, 64, 16, True, 8),
]


def run_select(logits, scores, done, take, eos, beam_major, ld_more=0):
    g, w, v = logits.shape
    lib = ph.library()
    flat = logits.reshape(g * w, v) if beam_major else logits.reshape(g * w, v).T
    buf = np.full((flat.shape[0], flat.shape[1] + ld_more), np.nan, np.float32)
    buf[:, :flat.shape[1]] = flat
    tl, ts, td = dev(buf), dev(scores), None if done is None else dev(done)
    need = lib.nnhip_beam_select_workspace_bytes(g, w, v, take)
    ws = torch.full((need // 4,), float("nan")).cuda()
    outs = []
    print(f"[select] groups {g} beams {w} vocab {v} take {take} beam_major {beam_major}", flush=True)
    for _ in range(2):
        out = [torch.full((g, take), -3.0).cuda() for _ in range(3)]
        assert lib.nnhip_beam_select(ptr(tl), buf.shape[1], int(beam_major), ptr(ts), ptr(td), g, w, v, take, eos,
                                     *[ptr(o) for o in out], ptr(ws), need, stream()) == 0
        outs.append(np.stack([o.cpu().numpy() for o in out]))
    assert np.array_equal(*outs)
    return outs[0]


def check_select(got, want):
    assert np.array_equal(got[1:], want[1:])
    fin = np.isfinite(want[0])
    assert np.array_equal(got[0][~fin], want[0][~fin])
    # the log-sum-exp is off by at most 2^-22 (each exp by 3 2^-24, each segment's sum by its 64 or 16 + 4
    # additions of terms that are no larger than it, in practice far less), the score by its own rounding
    assert np.all(np.abs(got[0][fin] - want[0][fin]) <= 70 * U + U * np.abs(want[0][fin]))


@pytest.mark.parametrize("groups,beams,vocab,take,beam_major,ended", SELECT)
@pytest.mark.parametrize("ld_more", [0, 5])
def test_select(groups, beams, vocab, take, beam_major, ended, ld_more):
    rng = np.random.default_rng(groups * 7 + beams * 13 + vocab)
    logits = rng.normal(0, 3, (groups, beams, vocab)).astype(np.float32)
    scores = rng.uniform(-30, 0, (groups, beams)).astype(np.float32)
    done = np.zeros((groups, beams), np.float32)
    for g in range(groups):
        done[g, rng.permutation(beams)[:ended]] = 1
    logits[done != 0] = np.nan         # never read
    eos = vocab // 2
    got = run_select(logits, scores, done if ended else None, take, eos, beam_major, ld_more)
    check_select(got, ph.select(logits, scores, done if ended else None, take, eos))


@pytest.mark.parametrize("beam_major", [False, True])
def test_select_many_groups(beam_major):
    """More beams than a launch has rows along its second axis."""
    g, w, v, take = 35001, 2, 37, 3
    rng = np.random.default_rng(5)
    logits = rng.normal(0, 3, (g, w, v)).astype(np.float32)
    scores = rng.uniform(-30, 0, (g, w)).astype(np.float32)
    check_select(run_select(logits, scores, None, take, 0, beam_major), ph.select(logits, scores, None, take, 0))


def test_select_scores_in_place():
    """out_score may be scores where as many are taken as there are beams."""
    g, w, v = 3, 7, 900
    rng = np.random.default_rng(6)
    logits = rng.normal(0, 3, (g, w, v)).astype(np.float32)
    scores = rng.uniform(-30, 0, (g, w)).astype(np.float32)
    want = run_select(logits, scores, None, w, 0, True)
    lib = ph.library()
    tl, ts = dev(logits.reshape(g * w, v)), dev(scores)
    need = lib.nnhip_beam_select_workspace_bytes(g, w, v, w)
    ws = torch.empty(need // 4, device="cuda")
    ob, ot = (torch.zeros(g, w).cuda() for _ in range(2))
    assert lib.nnhip_beam_select(ptr(tl), v, 1, ptr(ts), None, g, w, v, w, 0, ptr(ts), ptr(ob), ptr(ot), ptr(ws), need,
                                 stream()) == 0
    assert np.array_equal(np.stack([x.cpu().numpy() for x in (ts, ob, ot)]), want)


@pytest.mark.parametrize("beam_major", [False, True])
def test_select_ties(beam_major):
    """Equal totals in the order of beam, then token: all logits equal; two values; equal beams; no live beam."""
    g, w, v, take = 2, 6, 3001, 24
    rng = np.random.default_rng(1)
    same = np.zeros((g, w, v), np.float32)
    scores = np.full((g, w), -2.5, np.float32)
    got = run_select(same, scores, None, take, 0, beam_major)
    assert np.array_equal(got[2], np.tile(np.arange(take), (g, 1)))
    assert np.array_equal(got[1], np.array([[0] * take, [w] * take]))
    two = (rng.integers(0, 40, (g, w, v)) == 0).astype(np.float32)
    two[:] = two[:, :1]                # every beam of a group alike
    got = run_select(two, scores, None, take, 0, beam_major)
    check_select(got, ph.select(two, scores, None, take, 0))
    dead = np.full((g, w), -np.inf, np.float32)
    got = run_select(two, dead, None, take, 0, beam_major)
    assert np.all(got[0] == -np.inf) and np.array_equal(got[2], np.tile(np.arange(take), (g, 1)))


@pytest.mark.parametrize("beam_major", [False, True])
def test_select_odd_values(beam_major):
    """-inf logits are never taken before finite ones; a beam with NaN, with +inf or with nothing but -inf offers
    nothing; a first step with one live beam; more ended beams than live candidates."""
    g, w, v, take = 1, 6, 500, 12
    rng = np.random.default_rng(2)
    x = rng.normal(0, 2, (g, w, v)).astype(np.float32)
    x[0, 0, 7:] = -np.inf
    x[0, 1, 3] = np.nan
    x[0, 2, 9] = np.inf
    x[0, 3] = -np.inf
    x[0, 4, ::2] = -3.4028234663852886e38
    scores = np.array([[-1, 0, 0, 0, -4, -5]], np.float32)
    got = run_select(x, scores, None, take, 0, beam_major)
    check_select(got, ph.select(x, scores, None, take, 0))
    assert not set(got[1][0][np.isfinite(got[0][0])]) & {1, 2, 3}
    first = np.array([[0] + [-np.inf] * 5], np.float32)
    got = run_select(x, first, None, take, 0, beam_major)     # 7 finite candidates, then -inf ones by index
    check_select(got, ph.select(x, first, None, take, 0))
    done = np.array([[1, 1, 1, 1, 1, 0]], np.float32)
    x[0, 5, 2:] = -np.inf
    got = run_select(x, scores, done, take, 499, beam_major)
    check_select(got, ph.select(x, scores, done, take, 499))


# -- reordering ------------------------------------------------------------------
@pytest.mark.parametrize("batch,out_batch,page,layers,heads,dim,row_more", [
    (1, 1, 1, 1, 1, 1, 0), (4, 4, 1, 3, 2, 16, 0), (5, 8, 16, 2, 3, 20, 4), (8, 5, 7, 33, 1, 30, 1), (3, 3, 64, 2, 8, 128, 0),
    (6, 6, 24, 1, 12, 64, 0)])
@pytest.mark.parametrize("with_fresh", [True, False])
def test_reorder(batch, out_batch, page, layers, heads, dim, row_more, with_fresh):
    rng = np.random.default_rng(batch * 17 + page)
    width = 6
    pages = batch * width + 2 * out_batch
    perm = rng.permutation(pages).astype(np.float32)
    table = perm[:batch * width].reshape(batch, width)
    lens = rng.integers(0, width * page + 1, batch).astype(np.float32)
    lens[0] = width * page if batch > 1 else 2 * page + 1
    if batch > 2:
        lens[1], lens[2] = 2 * page, np.nan
        table[batch - 1, ph.length_of(lens[batch - 1], width * page) // page % width] = -1     # its page in progress is missing
    parent = rng.integers(0, batch, out_batch).astype(np.float32)
    fresh = perm[batch * width:batch * width + out_batch].copy()
    if out_batch > 2:
        parent[0], parent[out_batch - 1], fresh[1] = -1, batch, np.nan
    if out_batch > 3:
        p = int(parent[2])
        if ph.length_of(lens[p], width * page) // page < width:
            fresh[2] = table[p, ph.length_of(lens[p], width * page) // page]   # goes on in its parent's page
    row = heads * dim + row_more
    caches = [rng.normal(size=(pages * page, row)).astype(np.float32) for _ in range(2 * layers)]
    dv, tt = [dev(x) for x in caches], dev(table)
    c = dict(pages=pages, page=page, heads=heads, dim=dim, row=row)
    arr = (ph.Pages * layers)(*[cache(c, dv[2 * i], dv[2 * i + 1], tt) for i in range(layers)])
    tp, tl, tf = dev(parent), dev(lens), dev(fresh)
    out, n_out = torch.full((out_batch, width), 5.0).cuda(), torch.full((out_batch,), 5.0).cuda()
    print(f"[reorder] {batch} -> {out_batch} page {page} layers {layers}", flush=True)
    assert ph.library().nnhip_kv_reorder(arr, layers, ptr(tp), ptr(tl), ptr(tf) if with_fresh else None, out_batch, ptr(out),
                                         ptr(n_out), stream()) == 0
    w_out, w_n, w_c = ph.reorder([x[:, :heads * dim] for x in caches], table, page, pages, parent, lens,
                                 fresh if with_fresh else None, width)
    assert np.array_equal(out.cpu().numpy(), w_out, equal_nan=True) and np.array_equal(n_out.cpu().numpy(), w_n)
    for x, w, old in zip(dv, w_c, caches):
        assert np.array_equal(x.cpu().numpy()[:, :heads * dim], w)
        assert np.array_equal(x.cpu().numpy()[:, heads * dim:], old[:, heads * dim:])


# -- together --------------------------------------------------------------------
def test_captured_step_on_another_stream():
    """A step of a beam search (append, attention, selection, reordering) captured once and replayed with new inputs,
    eager work and synchronisation between the replays, against the same step run eagerly."""
    rng = np.random.default_rng(12)
    w, h, d, page, vocab, width = 5, 4, 32, 4, 999, 12
    B, f = w, h * d
    lib = ph.library()
    c = dict(pages=80, page=page, heads=h, dim=d)
    cos, sin = dev(np.cos(rng.uniform(0, 6, (48, d // 2)))), dev(np.sin(rng.uniform(0, 6, (48, d // 2))))
    table0 = np.full((B, width), -1.0, np.float32)
    table0[:, :5] = np.arange(5)
    table0[:, 5] = 10 + np.arange(B)
    st = dict(K=torch.zeros(80 * page, f).cuda(), V=torch.zeros(80 * page, f).cuda(), table=dev(table0),
              q=torch.zeros(f, B).cuda(), k=torch.zeros(f, B).cuda(), v=torch.zeros(f, B).cuda(),
              logits=torch.zeros(vocab, B).cuda(), scores=torch.zeros(B).cuda(), pos=torch.zeros(B).cuda(),
              lens=torch.zeros(B).cuda(), shared=dev([20.0]), fresh=dev(40 + np.arange(B)), qr=torch.zeros(f, B).cuda(),
              o=torch.zeros(f, B).cuda(), sel=torch.zeros(3, w).cuda(), tout=torch.zeros(B, width).cuda(),
              lout=torch.zeros(B).cuda())
    pg = cache(c, st["K"], st["V"], st["table"])
    n1, n2 = lib.nnhip_attn_paged_workspace_bytes(pg, h, w), lib.nnhip_beam_select_workspace_bytes(1, w, vocab, w)
    ws1, ws2 = torch.zeros(n1 // 4).cuda(), torch.zeros(n2 // 4).cuda()
    arr = (ph.Pages * 1)(pg)

    def step():
        s = stream()
        assert lib.nnhip_kv_append(pg, ptr(st["k"]), 1, B, ptr(st["v"]), 1, B, ptr(st["q"]), 1, B, ptr(st["qr"]), 1, B, h, B,
                                   None, ptr(st["pos"]), ptr(cos), ptr(sin), 48, d, s) == 0
        assert lib.nnhip_attn_paged(pg, ptr(st["qr"]), 1, B, h, ptr(st["lens"]), ptr(st["shared"]), w, None, 0.2,
                                    ptr(st["o"]), 1, B, None, None, ptr(ws1), n1, s) == 0
        assert lib.nnhip_beam_select(ptr(st["logits"]), B, 0, ptr(st["scores"]), None, 1, w, vocab, w, 0,
                                     *[ptr(x) for x in st["sel"]], ptr(ws2), n2, s) == 0
        assert lib.nnhip_kv_reorder(arr, 1, ptr(st["sel"][1]), ptr(st["lens"]), ptr(st["fresh"]), B, ptr(st["tout"]),
                                    ptr(st["lout"]), s) == 0

    def load(i):
        r = np.random.default_rng(100 + i)
        for n in ("q", "k", "v", "logits", "scores"):
            st[n].copy_(dev(r.normal(size=tuple(st[n].shape))))
        st["pos"].fill_(20.0 + i)
        st["lens"].fill_(21.0 + i)

    outs = ("K", "V", "qr", "o", "sel", "tout", "lout")
    base = {n: torch.randn_like(st[n]) for n in ("K", "V")}
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        load(0)
        step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
    torch.cuda.synchronize()
    for i in range(3):
        got = []
        for replay in (True, False):
            for n in ("K", "V"):
                st[n].copy_(base[n])
            load(i)
            torch.cuda.synchronize()
            if replay:
                graph.replay()
            else:
                step()
            torch.cuda.synchronize()
            got.append({n: st[n].clone() for n in outs})
        for n in outs:
            assert torch.equal(got[0][n], got[1][n]), (i, n)
