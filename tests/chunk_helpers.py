"""ctypes access to the 8-bit caches, chunk attention and draft verification (include/nnhip_kernels.h), and their plain
64-bit forms for the tests."""
import ctypes

import numpy as np

import paged_helpers as ph
from paged_helpers import LG, SZ, VP, Pages, index_of, length_of, row_of

U = 2.0 ** -24
LOWEST = -3.4028234663852886e38


class Pages8(ctypes.Structure):
    """nnhip_kv8_pages."""
    _fields_ = [(n, VP) for n in ("K", "V", "K_scale", "V_scale", "table")] + [
        (n, SZ) for n in ("batch", "width", "pages", "page", "heads", "dim", "row")]


def library():
    lib = ph.library()
    i32, f, pg, p8 = ctypes.c_int, ctypes.c_float, ctypes.POINTER(Pages), ctypes.POINTER(Pages8)
    lib.nnhip_kv8_append.argtypes = [p8, VP, LG, LG, VP, LG, LG, VP, LG, LG, VP, LG, LG, SZ, SZ, VP, VP, VP, VP, SZ, SZ, VP]
    lib.nnhip_kv8_read.argtypes = [p8, VP, LG, LG, VP, LG, LG, SZ, VP, VP, VP]
    for name, p in (("nnhip_attn_chunk", pg), ("nnhip_attn_chunk8", p8)):
        getattr(lib, name).argtypes = [p, VP, LG, LG, SZ, SZ, VP, SZ, VP, VP, f, VP, LG, LG, VP, VP, VP, SZ, VP]
        ws = getattr(lib, name + "_workspace_bytes")
        ws.argtypes, ws.restype = [p, SZ, SZ, SZ], SZ
    lib.nnhip_draft_verify.argtypes = [VP, SZ, VP, SZ, i32, SZ, SZ, VP, VP, SZ, SZ, f, VP, VP, VP, VP, VP, SZ, VP]
    lib.nnhip_draft_verify_workspace_bytes.argtypes = [SZ, SZ, SZ, SZ]
    lib.nnhip_draft_verify_workspace_bytes.restype = SZ
    return lib


# -- 8-bit caches ----------------------------------------------------------------
def turned(x, cos, sin, rope):
    """x (heads, dim) float32 by one position's cos and sin, in float64 (each product of two floats is exact there)."""
    y, h = x.astype(np.float64), rope // 2
    if h:
        a, b, co, si = y[:, :h].copy(), y[:, h:2 * h].copy(), cos.astype(np.float64), sin.astype(np.float64)
        with np.errstate(invalid="ignore", over="ignore"):
            y[:, :h], y[:, h:2 * h] = a * co - b * si, b * co + a * si
    return y


def quantise(y):
    """y (heads, dim) float64: bytes and scales (heads) as nnhip_kv8_append stores them."""
    scale, by = np.zeros(len(y), np.float32), np.zeros(y.shape, np.int8)
    for i, x in enumerate(y):
        if not np.all(np.isfinite(x)):
            scale[i] = np.nan
            continue
        scale[i] = np.float32(np.abs(x).max() / 127)
        if scale[i] > 0:
            by[i] = np.clip(np.rint(x / np.float64(scale[i])), -127, 127)
    return by, scale


def place(table, batch, page, pages, seq, pos, rope_rows, n):
    """Row and position of token n, None for padding."""
    b = n if seq is None else index_of(seq[n], batch)
    p = index_of(pos[n], 1 << 24)
    if b is None or b >= batch or p is None or (rope_rows and p >= rope_rows):
        return None, None
    return row_of(table, b, p, page, pages), p


# -- chunks of new tokens ----------------------------------------------------------
def attend(q, K, V, table, page, pages, heads, start, most, lens, alpha, slopes=None):
    """q (tokens, q_heads, dim); K, V (rows, heads, dim) float64: O, m, l, a bound on |O|'s error and one on m's, and which
    tokens belong to a sequence.

    The bound. A score is off by (dim + 4) 2^-24 times its terms' sizes for a chain of float32 products and additions (the
    bias and its subtraction twice more), and by 3 2^-24 of them where products are formed from two parts of 12 bits each
    (what two factors leave, 2^-24 each, and the product of their second parts); parts of values below 2^-29 of their
    row's largest end at 2^-39 of it. The exponent's argument is off by 2^-23 times the scores' size, exp2 by 2^-23, the
    factors that a range's and a wave's scores are scaled by alike. A weight is then off by twice the largest of these, the
    products with the values by another 3 2^-24, sums over n weights by n 2^-24 more, numerator and denominator alike, and
    weights below 2^-29 of the largest end at 2^-39 of the largest value."""
    N, H, D = q.shape
    B = len(lens)
    O, m, l = np.zeros((N, H, D)), np.full((N, H), LOWEST), np.zeros((N, H))
    tol, tol_m, has = np.zeros((N, H, D)), np.zeros((N, H)), np.zeros(N, bool)
    starts = [length_of(s, N) for s in start]
    for b in range(B):
        n = max(starts[b + 1] - starts[b], 0)
        size_of = length_of(lens[b], table.shape[1] * page)
        rows = [row_of(table, b, j, page, pages) for j in range(size_of)]
        there = np.array([j for j, r in enumerate(rows) if r is not None], dtype=np.int64)
        at = np.array([r for r in rows if r is not None], dtype=np.int64)
        for i in range(min(n, most)):
            t, p = starts[b] + i, size_of - n + i
            has[t] = True
            k = int(np.searchsorted(there, p + 1))   # positions up to p
            pos, r = there[:k], at[:k]
            if k == 0:
                continue
            for h in range(H):
                Kh, Vh, x = K[r, h * heads // H], V[r, h * heads // H], q[t, h].astype(np.float64)
                with np.errstate(invalid="ignore", over="ignore"):
                    s = alpha * (Kh @ x)
                    size = abs(alpha) * (np.abs(Kh) @ np.abs(x) * (1 + 7 * 2.0 ** -24) + D * 2.0 ** -14 * np.abs(Kh).max(1) * np.abs(x).max())
                    if slopes is not None:
                        s = s - slopes[h] * (p - pos)
                        size = size + 2 * abs(slopes[h]) * (p - pos)
                    if s.max() == -np.inf:
                        continue
                    m[t, h] = s.max()
                    w = np.exp(s - s.max())
                    l[t, h] = w.sum()
                    w = w / l[t, h]
                    O[t, h] = w @ Vh
                    err = (D + 7) * U * size.max()
                    tol_m[t, h] = err + 4 * U * np.abs(s).max()
                    off = 2 * (err + 4 * U * np.abs(s).max() + 4 * U) + (2 * k + 3) * U
                    tol[t, h] = 2 * off * (w @ np.abs(Vh)) + k * 2.0 ** -39 * np.abs(Vh).max(0) + 1e-30
    return O, m, l, tol, tol_m, has


# -- verification --------------------------------------------------------------------
def softmax64(z, temperature):
    z = np.where(np.isnan(z), -np.inf, z.astype(np.float64))
    m = z.max()
    if m == -np.inf:
        return np.zeros(len(z))
    with np.errstate(invalid="ignore", over="ignore"):
        e = np.where(z == m, 1.0, np.exp(np.where(z == m, 0.0, z - m) / temperature))
    return e / e.sum()


def verify(target, draft, fed, start, most, temperature, accept, pick):
    """target, draft (tokens, vocab): accepted and token of each sequence, and how near the random numbers came to a
    border, relative to it."""
    N, V = target.shape
    starts = [length_of(s, N) for s in start]
    accepted, token, near = [], [], np.inf
    for b in range(len(start) - 1):
        lo, n = starts[b], min(max(starts[b + 1] - starts[b], 0), most)
        if n == 0:
            accepted.append(0)
            token.append(-1)
            continue
        for i in range(n):
            x = index_of(fed[lo + i + 1], V) if i + 1 < n else None
            last = i + 1 == n
            if temperature == 0:
                z = np.where(np.isnan(target[lo + i]), -np.inf, target[lo + i])
                best = int(np.argmax(z))
                if not last and x == best:
                    continue
                token.append(best)
                break
            p = softmax64(target[lo + i], temperature)
            left = p
            if not last:
                if draft is None:
                    q = np.zeros(V)
                    if x is not None:
                        q[x] = 1.0
                else:
                    q = softmax64(draft[lo + i], temperature)
                u = float(accept[lo + i])
                if x is not None:
                    if p[x] > 0:
                        near = min(near, abs(u * q[x] / p[x] - 1))
                    if u * q[x] < p[x]:
                        continue
                left = np.maximum(p - q, 0)
                if left.sum() == 0:
                    left = p
            w = float(pick[b])
            w = 0.0 if not w > 0 else min(w, 1 - 2.0 ** -53)
            up = np.cumsum(left)
            if up[-1] == 0:
                token.append(0)
                break
            v = int(np.searchsorted(up, w * up[-1], side="right"))
            near = min(near, np.abs(up / up[-1] - w)[left > 0].min() if w > 0 and w < 1 - 1e-9 else np.inf)
            token.append(min(v, int(np.flatnonzero(left)[-1])))
            break
        accepted.append(i)
    return np.array(accepted), np.array(token), near
