"""ctypes access to the paged-cache and beam-search entry points (include/nnhip_kernels.h) for the tests."""
import ctypes

import numpy as np

import nnengine

SZ, LG, VP = ctypes.c_size_t, ctypes.c_long, ctypes.c_void_p


class Pages(ctypes.Structure):
    """nnhip_kv_pages."""
    _fields_ = [("K", VP), ("V", VP), ("table", VP)] + [
        (n, SZ) for n in ("batch", "width", "pages", "page", "heads", "dim", "row")]


def library():
    lib = nnengine.hip_library()
    pg, i32, f = ctypes.POINTER(Pages), ctypes.c_int, ctypes.c_float
    lib.nnhip_kv_append.argtypes = [pg, VP, LG, LG, VP, LG, LG, VP, LG, LG, VP, LG, LG, SZ, SZ, VP, VP, VP, VP, SZ, SZ, VP]
    lib.nnhip_attn_paged.argtypes = [pg, VP, LG, LG, SZ, VP, VP, SZ, VP, f, VP, LG, LG, VP, VP, VP, SZ, VP]
    lib.nnhip_attn_paged_workspace_bytes.argtypes = [pg, SZ, SZ]
    lib.nnhip_attn_paged_workspace_bytes.restype = SZ
    lib.nnhip_beam_select.argtypes = [VP, SZ, i32, VP, VP, SZ, SZ, SZ, SZ, SZ, VP, VP, VP, VP, SZ, VP]
    lib.nnhip_beam_select_workspace_bytes.argtypes = [SZ, SZ, SZ, SZ]
    lib.nnhip_beam_select_workspace_bytes.restype = SZ
    lib.nnhip_kv_reorder.argtypes = [pg, SZ, VP, VP, VP, SZ, VP, VP, VP]
    return lib


def index_of(x, limit):
    """A float-encoded index as the kernels read it: truncated toward zero, None outside [0, limit)."""
    x = float(x)
    if not x > -1.0 or not x < limit:
        return None
    return int(x)


def length_of(x, most):
    x = float(x)
    return 0 if not x >= 1.0 else int(min(x, most))


def row_of(table, b, pos, page, pages):
    i = pos // page
    if b >= table.shape[0] or i >= table.shape[1]:
        return None
    p = index_of(table[b, i], pages)
    return None if p is None else p * page + pos % page


def attend(q, K, V, table, page, pages, heads, lens, alpha, slopes=None):
    """q (batch, q_heads, dim); K, V (rows, heads, dim): O, m, l and a bound on |O|'s error in float32, all float64.

    The bound: scores off by at most (dim + 4) 2^-24 times the sum of their terms' sizes (each product and each
    addition of a chain rounds once, the bias and its subtraction twice more), as is the exponent's argument by
    2^-23 times the scores' size and exp2 by 2^-23 itself; a weight is then off by twice the largest of these, and
    the sums over n weights by n 2^-24 more, numerator and denominator alike."""
    B, H, D = q.shape
    O, m, l = np.zeros((B, H, D)), np.full((B, H), -3.4028234663852886e38), np.zeros((B, H))
    tol = np.zeros((B, H, D))
    u = 2.0 ** -24
    for b in range(B):
        n = length_of(lens[b], table.shape[1] * page)
        rows = [(j, row_of(table, b, j, page, pages)) for j in range(n)]
        pos = np.array([j for j, r in rows if r is not None], dtype=np.int64)
        if pos.size == 0:
            continue
        at = np.array([r for _, r in rows if r is not None])
        for h in range(H):
            k, v, x = K[at, h * heads // H], V[at, h * heads // H], q[b, h].astype(np.float64)
            with np.errstate(invalid="ignore", over="ignore"):
                s = alpha * (k @ x)
                size = abs(alpha) * (np.abs(k) @ np.abs(x))
                if slopes is not None:
                    s = s - slopes[h] * (n - 1 - pos)
                    size = size + 2 * abs(slopes[h]) * (n - 1 - pos)
                if s.max() == -np.inf:
                    continue
                m[b, h] = s.max()
                w = np.exp(s - s.max())
                l[b, h] = w.sum()
                O[b, h] = (w / l[b, h]) @ v
                off = 2 * ((D + 4) * u * size.max() + 4 * u * np.abs(s).max() + 4 * u) + 2 * pos.size * u
                tol[b, h] = 2 * off * ((w / l[b, h]) @ np.abs(v))
    return O, m, l, tol


def select(logits, scores, done, take, eos):
    """logits (groups, beams, vocab): scores, beams (over all groups) and tokens (groups, take) in float64."""
    g, w, v = logits.shape
    z = logits.astype(np.float64)
    with np.errstate(all="ignore"):
        m = z.max(axis=2, keepdims=True)
        lse = m + np.log(np.exp(z - m).sum(axis=2, keepdims=True))
        total = scores.astype(np.float64)[:, :, None] + (z - lse)
    if done is not None:
        for i, b in zip(*np.nonzero(done)):
            total[i, b] = -np.inf
            total[i, b, eos] = scores[i, b]
    total = np.where(np.isnan(total), -np.inf, total).reshape(g, w * v)
    out = np.empty((3, g, take))
    for i in range(g):
        at = np.lexsort((np.arange(w * v), -total[i]))[:take]
        out[:, i] = total[i, at], i * w + at // v, at % v
    return out


def reorder(caches, table, page, pages, parent, lens, fresh, width):
    """New tables, lengths and caches (copies) of nnhip_kv_reorder."""
    out = np.full((len(parent), width), -1.0)
    n_out = np.zeros(len(parent))
    new = [c.copy() for c in caches]
    for b, p in enumerate(parent):
        p = index_of(p, table.shape[0])
        if p is None:
            continue
        n = length_of(lens[p], width * page)
        full, tail = n // page, n % page
        n_out[b] = n
        out[b, :full] = table[p, :full]
        if full >= width:
            continue
        if fresh is None:
            out[b, full] = table[p, full] if tail else -1.0
            continue
        f = index_of(fresh[b], pages)
        out[b, full] = -1.0 if f is None else f
        src = index_of(table[p, full], pages)
        if f is None or src is None or f == src:
            continue
        for c, old in zip(new, caches):
            c[f * page:f * page + tail] = old[src * page:src * page + tail]
    return out, n_out, new
