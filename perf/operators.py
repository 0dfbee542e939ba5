"""Beam search over paged key/value caches: the operators' cases, plain forms and 64-bit results.

Each case calls one entry point of the kernel library (include/nnhip_kernels.h) on torch's tensors and stream:

  append   nnhip_kv_append: new tokens' keys and values into the pages, keys and queries rotated on the way
  attend   nnhip_attn_paged: one query a sequence against its pages, a group's shared prefix read once
  select   nnhip_beam_select: the best continuations of each group's beams over the vocabulary
  reorder  nnhip_kv_reorder: page tables by parent beam, the page in progress copied in every layer

Tensors are float32; index tensors hold integers as floats. With `own` false, run() computes the same from elementary
torch operations.
"""
import ctypes
import math
import os
import random
import sys

import numpy as np
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
own = False


# -- the cases ---------------------------------------------------------------
def listed():
    return [
        # One decoding step of a small beam search: 4 beams of a 768-wide model (12 heads of 64), rows of one token. The
        # smallest call: latency.
        dict(name="append_decode", kind="append", tokens=4, batch=4, q_heads=12, heads=12, dim=64, rope=64, page=1, past=300,
             feature_major=True, pad=0),
        # Five ragged prompts stored at once, grouped heads, pages of 64, some padding behind the last prompt.
        dict(name="append_prompts", kind="append", tokens=5003, batch=5, q_heads=32, heads=8, dim=128, rope=128, page=64,
             past=37, feature_major=False, pad=120),
        # 4 beams behind a prompt of 300 in the same model, ALiBi slopes: the smallest attention.
        dict(name="attend_small", kind="attend", groups=1, beams=4, q_heads=12, heads=12, dim=64, prefix=300, fresh=21,
             page=1, share=True, slopes=True, feature_major=True),
        # Four prompts of up to 1000 tokens (a context of 1024), 8 beams each.
        dict(name="attend_prompts", kind="attend", groups=4, beams=8, q_heads=12, heads=12, dim=64, prefix=1000, fresh=24,
             page=16, share=True, slopes=True, feature_major=True),
        # 16 samples of one long document, grouped heads.
        dict(name="attend_long", kind="attend", groups=1, beams=16, q_heads=32, heads=8, dim=128, prefix=65000, fresh=300,
             page=64, share=True, slopes=False, feature_major=False),
        # A served batch behind one instruction of 6000 tokens: 128 sequences, many rows to one key.
        dict(name="attend_batch", kind="attend", groups=1, beams=128, q_heads=32, heads=8, dim=128, prefix=6000, fresh=500,
             page=16, share=True, slopes=False, feature_major=False),
        # Nothing shared: 24 unrelated sequences of ragged lengths, an odd head width.
        dict(name="attend_apart", kind="attend", groups=24, beams=1, q_heads=8, heads=8, dim=80, prefix=5000, fresh=1,
             page=16, share=False, slopes=False, feature_major=False),
        # 4 beams over the small test model's 1024 classes: the smallest selection.
        dict(name="select_small", kind="select", groups=1, beams=4, vocab=1024, take=8, beam_major=False, first=False, ended=1),
        # 16 beams over the benchmark's 32000 classes, logits as the output head leaves them (vocabulary rows).
        dict(name="select_32000", kind="select", groups=1, beams=16, vocab=32000, take=32, beam_major=False, first=False,
             ended=2),
        # 32 prompts of 8 beams over a large vocabulary of odd size, a row of logits for each beam.
        dict(name="select_batch", kind="select", groups=32, beams=8, vocab=100003, take=16, beam_major=True, first=False,
             ended=1),
        # 4 beams, rows of one token: tables alone.
        dict(name="reorder_rows", kind="reorder", layers=12, batch=4, heads=12, dim=64, page=1, prefix=300, fresh=21),
        # 48 beams with pages of 32, the page in progress copied in 8 layers.
        dict(name="reorder_pages", kind="reorder", layers=8, batch=48, heads=8, dim=128, page=32, prefix=2000, fresh=50),
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "select", "select", "reorder"])
    heads = rng.choice([1, 2, 4, 8, 12])
    dim = rng.choice([16, 30, 32, 40, 64, 80, 96, 128])
    page = rng.choice([1, 8, 16, 24, 64])
    if kind == "append":
        tokens = _log(rng, 1, 4096)
        return dict(kind=kind, tokens=tokens, batch=rng.randint(1, min(tokens, 32)), q_heads=heads * rng.choice([1, 2, 4]),
                    heads=heads, dim=dim, rope=rng.choice([0, dim // 4 * 2, dim // 2 * 2]), page=page,
                    past=rng.randint(0, 2000), feature_major=rng.random() < 0.5, pad=rng.choice([0, 0, tokens // 3]))
    if kind == "attend":
        groups, beams = rng.choice([1, 1, 2, 4, 7]), _log(rng, 1, 64)
        return dict(kind=kind, groups=groups, beams=beams, q_heads=heads * rng.choice([1, 1, 2, 4]), heads=heads, dim=dim,
                    prefix=_log(rng, 1, 8000 if groups * beams <= 64 else 1500), fresh=_log(rng, 1, 200), page=page,
                    share=rng.random() < 0.8, slopes=rng.random() < 0.3, feature_major=rng.random() < 0.5)
    if kind == "select":
        groups, beams = _log(rng, 1, 16), _log(rng, 1, 32)
        vocab = _log(rng, 50, 60000)
        return dict(kind=kind, groups=groups, beams=beams, vocab=vocab, take=rng.randint(1, min(2 * beams, vocab)),
                    beam_major=rng.random() < 0.5, first=rng.random() < 0.2, ended=rng.randint(0, beams // 2))
    return dict(kind=kind, layers=rng.randint(1, 12), batch=_log(rng, 1, 32), heads=heads, dim=dim, page=page,
                prefix=_log(rng, 1, 1500), fresh=_log(rng, 1, 100))


# -- inputs ------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 29)


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * std


def _perm(g, n):
    return torch.randperm(n, generator=g, device="cuda")


def _sizes(c):
    """What a case fixes whatever the seed, tokens or lengths of each sequence: ragged where real batches are."""
    r = random.Random(len(c) * 7919 + c.get("batch", 0) + c.get("beams", 0))
    if c["kind"] == "append":
        n, b = c["tokens"] - c["pad"], c["batch"]
        cuts = sorted(r.randint(0, n) for _ in range(b - 1)) if n != b else list(range(1, b))
        count = [hi - lo for lo, hi in zip([0] + cuts, cuts + [n])]
        return dict(count=count, past=[r.randint(0, c["past"]) for _ in range(b)])
    if c["kind"] == "attend":
        prefix = [c["prefix"]] + [r.randint((c["prefix"] + 1) // 2, c["prefix"]) for _ in range(c["groups"] - 1)]
        own_ = [r.randint((c["fresh"] + 1) // 2, c["fresh"]) for _ in range(c["groups"] * c["beams"])]
        return dict(prefix=prefix, fresh=own_)
    return dict(len=c["prefix"] + c["fresh"])


def _rope_table(rows, rope):
    half = max(1, rope // 2)
    ang = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (
        -torch.arange(half, dtype=torch.float64, device="cuda") / half)
    return torch.cos(ang).float(), torch.sin(ang).float()


def _heads_tensor(c, g, n, heads):
    """(n, heads * dim) values, stored a token a row or a feature a row."""
    x = _randn(g, n, heads * c["dim"])
    return x.t().contiguous() if c["feature_major"] else x


def _append_inputs(c, seed):
    g, s = _gen(seed), _sizes(c)
    longest = max(n + p for n, p in zip(s["count"], s["past"]))
    width = (longest + c["page"] - 1) // c["page"]
    used = [(n + p + c["page"] - 1) // c["page"] for n, p in zip(s["count"], s["past"])]
    pages = sum(used) + 3
    table = torch.full((c["batch"], width), -1.0, device="cuda")
    at, order = 0, _perm(g, pages).float()
    for b, u in enumerate(used):
        table[b, :u] = order[at:at + u]
        at += u
    seq = [b for b, n in enumerate(s["count"]) for _ in range(n)] + [0] * c["pad"]
    pos = [p + i for n, p in zip(s["count"], s["past"]) for i in range(n)] + [-1] * c["pad"]
    k, v = (_heads_tensor(c, g, c["tokens"], c["heads"]) for _ in range(2))
    q = _heads_tensor(c, g, c["tokens"], c["q_heads"])
    cos, sin = _rope_table(longest, c["rope"])
    rows = pages * c["page"]
    K, V = (_randn(g, rows, c["heads"] * c["dim"]) for _ in range(2))
    return dict(K=K, V=V, table=table, pages=pages, k=k, v=v, q=q, out=torch.zeros_like(q), cos=cos, sin=sin,
                seq=torch.tensor(seq, dtype=torch.float32, device="cuda"),
                pos=torch.tensor(pos, dtype=torch.float32, device="cuda"))


def _attend_inputs(c, seed):
    g, s = _gen(seed), _sizes(c)
    p, w = c["page"], c["beams"]
    lens = [s["prefix"][b // w] + n for b, n in enumerate(s["fresh"])]
    # A group's sequences share whole pages; the page that the prefix ends in is each sequence's own.
    shared = [n // p * p if c["share"] else 0 for n in s["prefix"]]
    width = (max(lens) + p - 1) // p
    need = sum(n // p for n in shared) + sum((n + p - 1) // p - shared[b // w] // p for b, n in enumerate(lens))
    pages = need + 2
    order, table, at = _perm(g, pages).float(), torch.full((len(lens), width), -1.0, device="cuda"), 0
    for gr, n in enumerate(shared):
        table[gr * w:(gr + 1) * w, :n // p] = order[at:at + n // p]
        at += n // p
    for b, n in enumerate(lens):
        lo, hi = shared[b // w] // p, (n + p - 1) // p
        table[b, lo:hi] = order[at:at + hi - lo]
        at += hi - lo
    K, V = (_randn(g, pages * p, c["heads"] * c["dim"]) for _ in range(2))
    q = _heads_tensor(c, g, len(lens), c["q_heads"])
    f = dict(dtype=torch.float32, device="cuda")
    slopes = torch.tensor([2.0 ** (-8.0 * h / c["q_heads"]) for h in range(c["q_heads"])], **f) if c["slopes"] else None
    return dict(K=K, V=V, table=table, pages=pages, q=q, out=torch.empty_like(q), lens=torch.tensor(lens, **f),
                shared=torch.tensor(shared, **f), slopes=slopes)


def _select_inputs(c, seed):
    g = _gen(seed)
    n = c["groups"] * c["beams"]
    logits = _randn(g, n, c["vocab"], std=2.5)
    if not c["beam_major"]:
        logits = logits.t().contiguous()
    scores = -20.0 * torch.rand(c["groups"], c["beams"], generator=g, device="cuda")
    if c["first"]:   # the first step: one live beam a group
        scores[:, 1:] = -math.inf
    done = torch.zeros(c["groups"], c["beams"], device="cuda")
    if c["ended"]:
        done[:, -c["ended"]:] = 1.0
    return dict(logits=logits, scores=scores.reshape(-1).contiguous(), done=done.reshape(-1).contiguous(), eos=c["vocab"] // 3)


def _reorder_inputs(c, seed):
    g, s = _gen(seed), _sizes(c)
    p, b, n = c["page"], c["batch"], s["len"]
    shared = c["prefix"] // p
    used = (n + p - 1) // p
    width = used + 2
    pages = shared + b * (used - shared) + b
    order = _perm(g, pages).float()
    table = torch.full((b, width), -1.0, device="cuda")
    table[:, :shared] = order[:shared]
    table[:, shared:used] = order[shared:shared + b * (used - shared)].reshape(b, used - shared)
    caches = [_randn(g, pages * p, c["heads"] * c["dim"]) for _ in range(2 * c["layers"])]
    parent = torch.randint(0, b, (b,), generator=g, device="cuda").float()
    return dict(caches=caches, table=table, pages=pages, parent=parent, fresh=order[-b:].contiguous(),
                lens=torch.full((b,), float(n), device="cuda"), out=torch.zeros_like(table),
                out_len=torch.zeros(b, device="cuda"))


_INPUTS = dict(append=_append_inputs, attend=_attend_inputs, select=_select_inputs, reorder=_reorder_inputs)


class _Pages(ctypes.Structure):
    """nnhip_kv_pages."""
    _fields_ = [("K", ctypes.c_void_p), ("V", ctypes.c_void_p), ("table", ctypes.c_void_p)] + [
        (n, ctypes.c_size_t) for n in ("batch", "width", "pages", "page", "heads", "dim", "row")]


def _pages(c, x, K, V):
    return _Pages(K.data_ptr(), V.data_ptr(), x["table"].data_ptr(), x["table"].shape[0], x["table"].shape[1], x["pages"],
                  c["page"], c["heads"], c["dim"], c["heads"] * c["dim"])


def _strides(c, n, heads):
    """Floats from a token to the next and from a feature to the next."""
    return (1, n) if c["feature_major"] else (heads * c["dim"], 1)


def _library():
    sys.path.insert(0, os.path.join(ROOT, "neuralnet.cpp_amd"))
    import nnengine
    lib = nnengine.hip_library()
    vp, sz, lg, i32, f = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_long, ctypes.c_int, ctypes.c_float
    pg = ctypes.POINTER(_Pages)
    lib.nnhip_kv_append.argtypes = [pg, vp, lg, lg, vp, lg, lg, vp, lg, lg, vp, lg, lg, sz, sz, vp, vp, vp, vp, sz, sz, vp]
    lib.nnhip_attn_paged.argtypes = [pg, vp, lg, lg, sz, vp, vp, sz, vp, f, vp, lg, lg, vp, vp, vp, sz, vp]
    lib.nnhip_attn_paged_workspace_bytes.argtypes = [pg, sz, sz]
    lib.nnhip_attn_paged_workspace_bytes.restype = sz
    lib.nnhip_beam_select.argtypes = [vp, sz, i32, vp, vp, sz, sz, sz, sz, sz, vp, vp, vp, vp, sz, vp]
    lib.nnhip_beam_select_workspace_bytes.argtypes = [sz, sz, sz, sz]
    lib.nnhip_beam_select_workspace_bytes.restype = sz
    lib.nnhip_kv_reorder.argtypes = [pg, sz, vp, vp, vp, sz, vp, vp, vp]
    return lib


def prepare(case, seed):
    c = case
    x = _INPUTS[c["kind"]](c, seed)
    st = dict(case=c, x=x)
    if c["kind"] == "attend":
        # The lengths on the host, as the program that hands out the pages has them.
        st["lens"], st["shared"] = x["lens"].long().tolist(), x["shared"].long().tolist()
    return st


# -- one pass: the framework's calls -------------------------------------------
def _call(rc):
    if rc != 0:
        raise RuntimeError(f"the kernel library returned {rc}")


def _ws(st, lib, nbytes):
    if "ws" not in st:
        st["ws"] = torch.empty(max(1, nbytes // 4), device="cuda")
    return st["ws"].data_ptr(), 4 * st["ws"].numel()


def _lib_of(st):
    if "lib" not in st:
        st["lib"] = _library()
    return st["lib"]


def _own_append(st, c, x, stream):
    lib, n = _lib_of(st), c["tokens"]
    if "pg" not in st:
        st["pg"] = _pages(c, x, x["K"], x["V"])
    kv, qs = _strides(c, n, c["heads"]), _strides(c, n, c["q_heads"])
    rope = c["rope"] > 0
    _call(lib.nnhip_kv_append(st["pg"], x["k"].data_ptr(), *kv, x["v"].data_ptr(), *kv, x["q"].data_ptr(), *qs,
                              x["out"].data_ptr(), *qs, c["q_heads"], n, x["seq"].data_ptr(), x["pos"].data_ptr(),
                              x["cos"].data_ptr() if rope else None, x["sin"].data_ptr() if rope else None,
                              x["cos"].shape[0], c["rope"], stream))
    return [x["out"], x["K"], x["V"]]


def _own_attend(st, c, x, stream):
    lib, n = _lib_of(st), c["groups"] * c["beams"]
    if "pg" not in st:
        st["pg"] = _pages(c, x, x["K"], x["V"])
    ws = _ws(st, lib, lib.nnhip_attn_paged_workspace_bytes(st["pg"], c["q_heads"], c["beams"]) if "ws" not in st else 0)
    qs = _strides(c, n, c["q_heads"])
    _call(lib.nnhip_attn_paged(st["pg"], x["q"].data_ptr(), *qs, c["q_heads"], x["lens"].data_ptr(),
                               x["shared"].data_ptr() if c["share"] else None, c["beams"],
                               x["slopes"].data_ptr() if c["slopes"] else None, 1.0 / math.sqrt(c["dim"]),
                               x["out"].data_ptr(), *qs, None, None, *ws, stream))
    return [x["out"]]


def _own_select(st, c, x, stream):
    lib = _lib_of(st)
    g, w, v, k = c["groups"], c["beams"], c["vocab"], c["take"]
    if "out" not in st:
        st["out"] = [torch.empty(g, k, device="cuda") for _ in range(3)]
    ws = _ws(st, lib, lib.nnhip_beam_select_workspace_bytes(g, w, v, k) if "ws" not in st else 0)
    _call(lib.nnhip_beam_select(x["logits"].data_ptr(), v if c["beam_major"] else g * w, int(c["beam_major"]),
                                x["scores"].data_ptr(), x["done"].data_ptr(), g, w, v, k, x["eos"],
                                *[t.data_ptr() for t in st["out"]], *ws, stream))
    return st["out"]


def _own_reorder(st, c, x, stream):
    lib = _lib_of(st)
    if "pg" not in st:
        st["pg"] = (_Pages * c["layers"])(*[_pages(c, x, x["caches"][2 * i], x["caches"][2 * i + 1])
                                            for i in range(c["layers"])])
    _call(lib.nnhip_kv_reorder(st["pg"], c["layers"], x["parent"].data_ptr(), x["lens"].data_ptr(), x["fresh"].data_ptr(),
                               c["batch"], x["out"].data_ptr(), x["out_len"].data_ptr(), stream))
    return [x["out"], x["out_len"]] + x["caches"]


# -- one pass: the plain forms -------------------------------------------------
def _tokens(c, x):
    """(n, features) view of a tensor stored either way."""
    return x.t() if c["feature_major"] else x


def _row_index(c, table, seq, pos):
    return table[seq, torch.div(pos, c["page"], rounding_mode="floor")].long() * c["page"] + pos % c["page"]


def _rotate(c, x, cos, sin):
    """x (n, heads, dim) with features j and j + rope/2 of each head turned by the token's angles."""
    h = c["rope"] // 2
    if h == 0:
        return x
    a, b, co, si = x[..., :h], x[..., h:2 * h], cos[:, None, :h], sin[:, None, :h]
    return torch.cat([a * co - b * si, b * co + a * si, x[..., 2 * h:]], dim=2)


def _plain_append(st, c, x):
    live = torch.nonzero(x["pos"] >= 0)[:, 0]
    seq, pos = x["seq"][live].long(), x["pos"][live].long()
    rows = _row_index(c, x["table"], seq, pos)
    cos, sin = x["cos"][pos], x["sin"][pos]
    k = _tokens(c, x["k"])[live].reshape(-1, c["heads"], c["dim"])
    q = _tokens(c, x["q"])[live].reshape(-1, c["q_heads"], c["dim"])
    x["K"][rows] = _rotate(c, k, cos, sin).reshape(len(live), -1)
    x["V"][rows] = _tokens(c, x["v"])[live]
    _tokens(c, x["out"])[live] = _rotate(c, q, cos, sin).reshape(len(live), -1)
    return [x["out"], x["K"], x["V"]]


def _scores(c, q, K):
    """alpha q k: q (heads, rows, dim), K (heads, n, dim) -> (heads, rows, n)."""
    return torch.matmul(q, K.transpose(1, 2).contiguous()) * (1.0 / math.sqrt(c["dim"]))


def _plain_group(c, x, b0, w, longest, shared):
    """Sequences b0 .. b0 + w - 1, whose first `shared` positions are the same rows."""
    d, kh, r = c["dim"], c["heads"], c["q_heads"] // c["heads"]
    q = _tokens(c, x["q"])[b0:b0 + w].reshape(w, kh, r, d).permute(1, 0, 2, 3)            # (kv heads, beams, r, d)
    pre = torch.arange(shared, device="cuda")
    rows = _row_index(c, x["table"], b0, pre)
    slopes = None if x["slopes"] is None else x["slopes"].reshape(kh, 1, r, 1)
    last = x["lens"][b0:b0 + w] - 1
    m = longest - shared
    # The prefix: one product for all of the group's rows.
    Kp, Vp = (x[n][rows].reshape(shared, kh, d).permute(1, 0, 2).contiguous() for n in ("K", "V"))
    sp = _scores(c, q.reshape(kh, w * r, d), Kp).reshape(kh, w, r, shared)
    # Each sequence's own positions, padded to the longest.
    pos = shared + torch.arange(m, device="cuda")
    there = pos[None, :] < x["lens"][b0:b0 + w, None]
    at = torch.where(there, pos[None, :], 0)
    own_rows = _row_index(c, x["table"], torch.arange(b0, b0 + w, device="cuda")[:, None], at)
    Ko, Vo = (x[n][own_rows].reshape(w, m, kh, d).permute(2, 0, 1, 3).reshape(kh * w, m, d).contiguous() for n in ("K", "V"))
    so = _scores(c, q.reshape(kh * w, r, d), Ko).reshape(kh, w, r, m)
    if slopes is not None:
        sp = sp - slopes * (last[None, :, None, None] - pre)
        so = so - slopes * (last[None, :, None, None] - pos)
    so = torch.where(there[None, :, None, :], so, -math.inf)
    top = so.amax(3, keepdim=True)
    if shared:
        top = torch.maximum(top, sp.amax(3, keepdim=True))
    ep, eo = torch.exp(sp - top), torch.exp(so - top)
    total = ep.sum(3, keepdim=True) + eo.sum(3, keepdim=True)
    o = torch.matmul(ep.reshape(kh, w * r, shared), Vp).reshape(kh, w, r, d)
    o = o + torch.matmul(eo.reshape(kh * w, r, m), Vo).reshape(kh, w, r, d)
    return (o / total).permute(1, 0, 2, 3).reshape(w, -1)


def _plain_attend(st, c, x):
    w = c["beams"]
    if c["share"]:
        out = torch.cat([_plain_group(c, x, g * w, w, max(st["lens"][g * w:(g + 1) * w]), n)
                         for g, n in enumerate(st["shared"])])
    else:
        out = _plain_group(c, x, 0, len(st["lens"]), max(st["lens"]), 0)
    return [out.t().contiguous() if c["feature_major"] else out]


def _plain_select(st, c, x):
    g, w, v, k = c["groups"], c["beams"], c["vocab"], c["take"]
    z = (x["logits"] if c["beam_major"] else x["logits"].t()).double()
    z = z - z.amax(1, keepdim=True)
    logp = z - torch.log(torch.exp(z).sum(1, keepdim=True))
    token = torch.arange(v, device="cuda")[None, :]
    ended = torch.where(token == x["eos"], 0.0, -math.inf).double()
    total = x["scores"].double()[:, None] + torch.where(x["done"][:, None] != 0, ended, logp)
    total, at = torch.sort(total.reshape(g, w * v), dim=1, descending=True, stable=True)
    at = at[:, :k]
    beam = torch.arange(g, device="cuda")[:, None] * w + torch.div(at, v, rounding_mode="floor")
    return [total[:, :k].float(), beam.float(), (at % v).float()]


def _plain_reorder(st, c, x):
    p, n = c["page"], int(_sizes(c)["len"])
    parent, full, tail = x["parent"].long(), n // p, n % p
    out = torch.full_like(x["table"], -1.0)
    out[:, :full] = x["table"][parent, :full]
    out[:, full] = x["fresh"]
    if tail:
        i = torch.arange(tail, device="cuda")
        src = (x["table"][parent, full].long()[:, None] * p + i).reshape(-1)
        dst = (x["fresh"].long()[:, None] * p + i).reshape(-1)
        for t in x["caches"]:
            t[dst] = t[src]
    return [out, x["lens"][parent]] + x["caches"]


def run(state):
    c, x = state["case"], state["x"]
    if own:
        stream = torch.cuda.current_stream().cuda_stream
        return {"append": _own_append, "attend": _own_attend, "select": _own_select,
                "reorder": _own_reorder}[c["kind"]](state, c, x, stream)
    return {"append": _plain_append, "attend": _plain_attend, "select": _plain_select,
            "reorder": _plain_reorder}[c["kind"]](state, c, x)


# -- what a pass cannot do without -------------------------------------------
def work(case):
    c, s = case, _sizes(case) if case["kind"] != "select" else None
    if c["kind"] == "append":
        n = c["tokens"] - c["pad"]
        values = n * c["dim"] * (2 * c["heads"] + c["q_heads"])
        turned = n * c["rope"] * (c["heads"] + c["q_heads"])
        return dict(bytes=8.0 * values + 4.0 * n * (c["rope"] + 3), flops=3.0 * turned)
    if c["kind"] == "attend":
        w, p = c["beams"], c["page"]
        lens = [s["prefix"][b // w] + n for b, n in enumerate(s["fresh"])]
        shared = [n // p * p if c["share"] else 0 for n in s["prefix"]]
        rows = sum(shared) + sum(n - shared[b // w] for b, n in enumerate(lens))
        return dict(bytes=8.0 * c["dim"] * (rows * c["heads"] + len(lens) * c["q_heads"]) + 4.0 * rows / p,
                    flops=4.0 * c["dim"] * c["q_heads"] * sum(lens))
    if c["kind"] == "select":
        n = c["groups"] * c["beams"]
        return dict(bytes=4.0 * (n - c["groups"] * c["ended"]) * c["vocab"] + 8.0 * n + 12.0 * c["groups"] * c["take"],
                    flops=5.0 * n * c["vocab"])
    rows = c["batch"] * (s["len"] % c["page"])
    table = c["batch"] * ((s["len"] + c["page"] - 1) // c["page"] + 2)
    return dict(bytes=8.0 * rows * c["heads"] * c["dim"] * 2 * c["layers"] + 8.0 * table + 16.0 * c["batch"], flops=0.0)


# -- the same results in 64 bits ---------------------------------------------
def _exact_append(c, x):
    tok = lambda t, h: (t.T if c["feature_major"] else t).double().reshape(c["tokens"], h, c["dim"])  # noqa: E731
    half = c["rope"] // 2
    out, K, V = x["out"].double(), x["K"].double(), x["V"].double()
    at = [n for n, p in enumerate(x["pos"].tolist()) if p >= 0]
    pos, seq = x["pos"].long()[at], x["seq"].long()[at]
    row = x["table"].long()[seq, pos // c["page"]] * c["page"] + pos % c["page"]

    def turned(z):
        z = z.clone()
        if half:
            # a pair as a complex number times e^(i angle)
            w = torch.complex(z[..., :half], z[..., half:2 * half]) * torch.complex(
                x["cos"].double()[pos], x["sin"].double()[pos])[:, None, :]
            z[..., :half], z[..., half:2 * half] = w.real, w.imag
        return z.reshape(len(at), -1)

    K[row], V[row] = turned(tok(x["k"], c["heads"])[at]), tok(x["v"], c["heads"])[at].reshape(len(at), -1)
    (out.T if c["feature_major"] else out)[at] = turned(tok(x["q"], c["q_heads"])[at])
    return [out, K, V]


def _exact_attend(c, x):
    r, d = c["q_heads"] // c["heads"], c["dim"]
    q = (x["q"].T if c["feature_major"] else x["q"]).double().reshape(-1, c["heads"], r, d)
    out = []
    for b, n in enumerate(x["lens"].long().tolist()):
        j = torch.arange(n, device="cuda")
        row = x["table"][b].long()[j // c["page"]] * c["page"] + j % c["page"]
        K, V = (x[t][row].double().reshape(n, c["heads"], d).transpose(0, 1).contiguous() for t in ("K", "V"))
        s = (K @ q[b].transpose(1, 2).contiguous()) / math.sqrt(d)                        # (heads, n, r)
        if x["slopes"] is not None:
            s = s - x["slopes"].double().reshape(c["heads"], 1, r) * (n - 1 - j)[None, :, None]
        s = torch.softmax(s, dim=1)
        out.append((s.transpose(1, 2).contiguous() @ V).reshape(-1))
    out = torch.stack(out)
    return [out.T.contiguous() if c["feature_major"] else out]


def _exact_select(c, x):
    g, w, v, k = c["groups"], c["beams"], c["vocab"], c["take"]
    z = (x["logits"] if c["beam_major"] else x["logits"].T).double()
    total = z - torch.logsumexp(z, 1, keepdim=True) + x["scores"].double()[:, None]
    for b in torch.nonzero(x["done"])[:, 0].tolist():
        total[b] = -math.inf
        total[b, x["eos"]] = x["scores"].double()[b]
    total = total.reshape(g, w * v).cpu().numpy()
    out = np.empty((3, g, k))
    for i, row in enumerate(total):
        kth = np.partition(row, len(row) - k)[len(row) - k]
        at = np.nonzero(row >= kth)[0]
        at = at[np.lexsort((at, -row[at]))][:k]
        out[:, i] = row[at], i * w + at // v, at % v
    return [torch.from_numpy(t) for t in out]


def _exact_reorder(c, x):
    p, n = c["page"], _sizes(c)["len"]
    table, fresh = x["table"].cpu().numpy(), x["fresh"].cpu().numpy()
    out = np.full_like(table, -1.0)
    moves = []
    for b, par in enumerate(int(i) for i in x["parent"].tolist()):
        for i in range(n // p + 1):
            out[b, i] = table[par, i] if i < n // p else fresh[b]
        moves += [(int(fresh[b]) * p + i, int(table[par, n // p]) * p + i) for i in range(n % p)]
    caches = [t.double() for t in x["caches"]]
    if moves:
        dst, src = (torch.tensor(m, device="cuda") for m in zip(*moves))
        for t in caches:
            t.index_copy_(0, dst, t.index_select(0, src))
    return [torch.from_numpy(out).double(), x["lens"].double()] + caches


def exact(case, seed):
    x = _INPUTS[case["kind"]](case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "select": _exact_select,
            "reorder": _exact_reorder}[case["kind"]](case, x)
