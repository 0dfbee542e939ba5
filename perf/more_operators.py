"""Drafted tokens over paged caches, in float32 and in 8 bits: the operators' cases, plain forms and 64-bit results.

Each case calls entry points of the kernel library (include/nnhip_kernels.h) on torch's tensors and stream:

  store   nnhip_kv8_append, then nnhip_kv8_read of the same tokens: keys and values quantised as they are written, keys and
          queries rotated on the way, and what the cache stands for
  read    nnhip_kv8_read: whole sequences out of an 8-bit cache
  chunk   nnhip_attn_chunk (bits 32) or nnhip_attn_chunk8 (bits 8): each sequence's new tokens against its pages
  verify  nnhip_draft_verify: how many drafted tokens stand, and the token behind them

Tensors are float32, but for the bytes of 8-bit caches; index tensors hold integers as floats. With `own` false, run()
computes the same from elementary torch operations.
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
        # One step of four sequences of a 768-wide model (12 heads of 64), a token each: the smallest call, latency.
        dict(name="store_decode", kind="store", tokens=4, batch=4, q_heads=12, heads=12, dim=64, rope=64, page=1, past=300,
             feature_major=True, pad=0),
        # Five ragged prompts stored at once, grouped heads, pages of 64, some padding behind the last prompt.
        dict(name="store_prompts", kind="store", tokens=4999, batch=5, q_heads=32, heads=8, dim=128, rope=128, page=64,
             past=37, feature_major=False, pad=101),
        # One sequence of 321 positions, rows of one token, out of the small model's cache.
        dict(name="read_small", kind="read", batch=1, heads=12, dim=64, page=1, longest=321, feature_major=True),
        # Nine sequences of up to 5000 positions, to go on in float32 pages.
        dict(name="read_long", kind="read", batch=9, heads=8, dim=128, page=16, longest=5000, feature_major=False),
        # Four drafted tokens and the one before them behind 700 positions, 12 heads of 64, ALiBi: latency.
        dict(name="chunk_verify", kind="chunk", bits=32, batch=1, new=5, mix="same", past=700, q_heads=12, heads=12, dim=64,
             page=16, slopes=True, feature_major=True),
        # A served batch: one prompt of 517 tokens beside 31 sequences that take one token each.
        dict(name="chunk_mixed", kind="chunk", bits=32, batch=32, new=517, mix="one", past=3000, q_heads=12, heads=12, dim=64,
             page=16, slopes=False, feature_major=True),
        # 2048 tokens of a long prompt behind 6000, grouped heads: the largest.
        dict(name="chunk_prompt", kind="chunk", bits=32, batch=1, new=2048, mix="same", past=6000, q_heads=32, heads=8, dim=128,
             page=64, slopes=False, feature_major=False),
        # 48 sequences of up to 8000 positions, a token each, over an 8-bit cache.
        dict(name="chunk8_decode", kind="chunk", bits=8, batch=48, new=1, mix="same", past=8000, q_heads=32, heads=8, dim=128,
             page=16, slopes=False, feature_major=False),
        # Ragged chunks of up to 1000 tokens of seven prompts over an 8-bit cache, an odd head width.
        dict(name="chunk8_prompts", kind="chunk", bits=8, batch=7, new=1000, mix="ragged", past=4000, q_heads=16, heads=8,
             dim=80, page=16, slopes=False, feature_major=False),
        # Four drafted tokens over the small test model's 1024 classes: the smallest verification.
        dict(name="verify_small", kind="verify", batch=1, drafted=4, vocab=1024, token_major=False, temperature=1.0, draft=True),
        # 24 sequences of up to five drafted tokens over the benchmark's 32000 classes, logits as the output head leaves them.
        dict(name="verify_32000", kind="verify", batch=24, drafted=5, vocab=32000, token_major=False, temperature=0.8,
             draft=True),
        # 32 sequences of up to seven over a large vocabulary of odd size, a row of logits a token.
        dict(name="verify_batch", kind="verify", batch=32, drafted=7, vocab=100003, token_major=True, temperature=1.0,
             draft=True),
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "read", "chunk", "chunk", "chunk", "chunk", "verify", "verify"])
    heads = rng.choice([1, 2, 4, 8, 12])
    dim = rng.choice([16, 30, 32, 40, 64, 80, 96, 128])
    page = rng.choice([1, 8, 16, 24, 64])
    if kind == "store":
        tokens = _log(rng, 1, 4096)
        return dict(kind=kind, tokens=tokens, batch=rng.randint(1, min(tokens, 32)), q_heads=heads * rng.choice([1, 2, 4]),
                    heads=heads, dim=dim, rope=rng.choice([0, dim // 4 * 2, dim // 2 * 2]), page=page,
                    past=rng.randint(0, 2000), feature_major=rng.random() < 0.5, pad=rng.choice([0, 0, tokens // 3]))
    if kind == "read":
        return dict(kind=kind, batch=_log(rng, 1, 16), heads=heads, dim=dim, page=page, longest=_log(rng, 1, 3000),
                    feature_major=rng.random() < 0.5)
    if kind == "chunk":
        new = _log(rng, 1, 1024)
        case = dict(kind=kind, bits=rng.choice([32, 8]), batch=_log(rng, 1, 32) if new <= 64 else rng.randint(1, 4), new=new,
                    mix=rng.choice(["same", "one", "ragged"]), past=_log(rng, 1, 6000) - 1, q_heads=heads * rng.choice([1, 1, 2, 4]),
                    heads=heads, dim=dim, page=page, slopes=rng.random() < 0.3, feature_major=rng.random() < 0.5)
        while work(case)["flops"] > 2e11:   # the largest listed one has 2.4e11
            case["batch"], case["past"] = (case["batch"] + 1) // 2, case["past"] // 2
        return case
    return dict(kind=kind, batch=_log(rng, 1, 32), drafted=rng.randint(0, 8), vocab=_log(rng, 50, 60000),
                token_major=rng.random() < 0.5, temperature=rng.choice([0.0, 0.7, 1.0, 1.3]), draft=rng.random() < 0.8)


# -- inputs ------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 31)


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * std


def _f(values):
    return torch.tensor(values, dtype=torch.float32, device="cuda")


def _sizes(c):
    """What a case fixes whatever the seed: the tokens and positions of each sequence, ragged where real batches are."""
    r = random.Random(len(c) * 7919 + c["batch"] * 31 + c.get("new", 0) + c.get("drafted", 0))
    if c["kind"] == "store":
        n, b = c["tokens"] - c["pad"], c["batch"]
        cuts = sorted(r.randint(0, n) for _ in range(b - 1)) if n != b else list(range(1, b))
        return dict(count=[hi - lo for lo, hi in zip([0] + cuts, cuts + [n])], past=[r.randint(0, c["past"]) for _ in range(b)])
    if c["kind"] == "read":
        return dict(len=[c["longest"]] + [r.randint((c["longest"] + 1) // 2, c["longest"]) for _ in range(c["batch"] - 1)])
    if c["kind"] == "verify":
        return dict(count=[c["drafted"] + 1] + [r.randint(1, c["drafted"] + 1) for _ in range(c["batch"] - 1)])
    new = {"same": lambda i: c["new"], "one": lambda i: c["new"] if i == c["batch"] // 3 else 1,
           "ragged": lambda i: c["new"] if i == 0 else r.randint((c["new"] + 1) // 2, c["new"])}[c["mix"]]
    past = [c["past"]] + [r.randint((c["past"] + 1) // 2, c["past"]) for _ in range(c["batch"] - 1)]
    return dict(count=[new(i) for i in range(c["batch"])], past=past)


def _starts(count):
    return [0] + [int(n) for n in np.cumsum(count)]


def _rope_table(rows, rope):
    half = max(1, rope // 2)
    ang = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (
        -torch.arange(half, dtype=torch.float64, device="cuda") / half)
    return torch.cos(ang).float(), torch.sin(ang).float()


def _heads_tensor(c, g, n, heads):
    """(n, heads * dim) values, stored a token a row or a feature a row."""
    x = _randn(g, n, heads * c["dim"])
    return x.t().contiguous() if c["feature_major"] else x


def _page_table(c, g, lens, spare):
    """Pages handed out in random order, -1 behind each sequence's last."""
    page = c["page"]
    used = [(n + page - 1) // page for n in lens]
    pages = sum(used) + spare
    order = torch.randperm(pages, generator=g, device="cuda").float()
    table, at = torch.full((len(lens), max(1, max(used))), -1.0, device="cuda"), 0
    for b, u in enumerate(used):
        table[b, :u] = order[at:at + u]
        at += u
    return table, pages


def _bytes_cache(c, g, rows):
    """An 8-bit cache as appending leaves it: every head's row has a byte of 127 or -127, scales around 3 / 127."""
    x = _randn(g, rows, c["heads"], c["dim"])
    top = x.abs().amax(2, keepdim=True)
    scale = (top / 127 * torch.exp(_randn(g, rows, c["heads"], 1, std=0.3)))[..., 0].contiguous()
    return torch.round(x / top * 127).to(torch.int8).reshape(rows, -1), scale


def _store_inputs(c, seed):
    g, s = _gen(seed), _sizes(c)
    lens = [n + p for n, p in zip(s["count"], s["past"])]
    table, pages = _page_table(c, g, lens, 3)
    seq = [b for b, n in enumerate(s["count"]) for _ in range(n)] + [0] * c["pad"]
    pos = [p + i for n, p in zip(s["count"], s["past"]) for i in range(n)] + [-1] * c["pad"]
    k, v = (_heads_tensor(c, g, c["tokens"], c["heads"]) for _ in range(2))
    q = _heads_tensor(c, g, c["tokens"], c["q_heads"])
    cos, sin = _rope_table(max(lens), c["rope"])
    rows = pages * c["page"]
    K, Ks = _bytes_cache(c, g, rows)
    V, Vs = _bytes_cache(c, g, rows)
    return dict(K=K, V=V, Ks=Ks, Vs=Vs, table=table, pages=pages, k=k, v=v, q=q, out=torch.zeros_like(q),
                k_back=torch.zeros_like(k), v_back=torch.zeros_like(v), cos=cos, sin=sin, seq=_f(seq), pos=_f(pos))


def _read_inputs(c, seed):
    g, s = _gen(seed), _sizes(c)
    table, pages = _page_table(c, g, s["len"], 3)
    K, Ks = _bytes_cache(c, g, pages * c["page"])
    V, Vs = _bytes_cache(c, g, pages * c["page"])
    n = sum(s["len"])
    shape = (c["heads"] * c["dim"], n) if c["feature_major"] else (n, c["heads"] * c["dim"])
    return dict(K=K, V=V, Ks=Ks, Vs=Vs, table=table, pages=pages, k_back=torch.zeros(shape, device="cuda"),
                v_back=torch.zeros(shape, device="cuda"), seq=_f([b for b, m in enumerate(s["len"]) for _ in range(m)]),
                pos=_f([i for m in s["len"] for i in range(m)]))


def _chunk_inputs(c, seed):
    g, s = _gen(seed), _sizes(c)
    lens = [n + p for n, p in zip(s["count"], s["past"])]
    table, pages = _page_table(c, g, lens, 2)
    rows, n = pages * c["page"], sum(s["count"])
    x = dict(table=table, pages=pages, start=_f(_starts(s["count"])), lens=_f(lens))
    if c["bits"] == 8:
        x["K"], x["Ks"] = _bytes_cache(c, g, rows)
        x["V"], x["Vs"] = _bytes_cache(c, g, rows)
    else:
        x["K"], x["V"] = (_randn(g, rows, c["heads"] * c["dim"]) for _ in range(2))
    x["q"] = _heads_tensor(c, g, n, c["q_heads"])
    x["out"] = torch.empty_like(x["q"])
    x["slopes"] = _f([2.0 ** (-8.0 * (h + 1) / c["q_heads"]) for h in range(c["q_heads"])]) if c["slopes"] else None
    return x


def _verify_inputs(c, seed):
    """The draft's logits are the target's and noise; drafted tokens are drawn from the draft's distribution."""
    g, s = _gen(seed), _sizes(c)
    n = sum(s["count"])
    target = _randn(g, n, c["vocab"], std=2.5)
    draft = target + _randn(g, n, c["vocab"], std=0.5)
    noise = -torch.log(-torch.log(torch.rand(n, c["vocab"], generator=g, device="cuda").clamp(1e-7, 1 - 1e-7)))
    drawn = (draft / c["temperature"] + noise if c["temperature"] > 0 else draft).argmax(1)
    fed = torch.zeros(n, device="cuda")
    fed[1:] = drawn[:-1].float()   # row i's token is the next row's
    first = torch.tensor(_starts(s["count"])[:-1], device="cuda")
    fed[first] = torch.randint(0, c["vocab"], (len(first),), generator=g, device="cuda").float()
    if not c["token_major"]:
        target, draft = target.t().contiguous(), draft.t().contiguous()
    return dict(target=target, draft=draft if c["draft"] else None, fed=fed, start=_f(_starts(s["count"])),
                accept=torch.rand(n, generator=g, device="cuda"), pick=torch.rand(c["batch"], generator=g, device="cuda"))


_INPUTS = dict(store=_store_inputs, read=_read_inputs, chunk=_chunk_inputs, verify=_verify_inputs)


class _Pages(ctypes.Structure):
    """nnhip_kv_pages."""
    _fields_ = [("K", ctypes.c_void_p), ("V", ctypes.c_void_p), ("table", ctypes.c_void_p)] + [
        (n, ctypes.c_size_t) for n in ("batch", "width", "pages", "page", "heads", "dim", "row")]


class _Pages8(ctypes.Structure):
    """nnhip_kv8_pages."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("K", "V", "K_scale", "V_scale", "table")] + [
        (n, ctypes.c_size_t) for n in ("batch", "width", "pages", "page", "heads", "dim", "row")]


def _pages(c, x):
    sizes = (x["table"].shape[0], x["table"].shape[1], x["pages"], c["page"], c["heads"], c["dim"], c["heads"] * c["dim"])
    if "Ks" in x:
        return _Pages8(*[x[n].data_ptr() for n in ("K", "V", "Ks", "Vs", "table")], *sizes)
    return _Pages(*[x[n].data_ptr() for n in ("K", "V", "table")], *sizes)


def _strides(c, n, heads):
    """Floats from a token to the next and from a feature to the next."""
    return (1, n) if c["feature_major"] else (heads * c["dim"], 1)


def _library():
    sys.path.insert(0, os.path.join(ROOT, "neuralnet.cpp_amd"))
    import nnengine
    lib = nnengine.hip_library()
    vp, sz, lg, i32, f = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_long, ctypes.c_int, ctypes.c_float
    pg, p8 = ctypes.POINTER(_Pages), ctypes.POINTER(_Pages8)
    lib.nnhip_kv8_append.argtypes = [p8, vp, lg, lg, vp, lg, lg, vp, lg, lg, vp, lg, lg, sz, sz, vp, vp, vp, vp, sz, sz, vp]
    lib.nnhip_kv8_read.argtypes = [p8, vp, lg, lg, vp, lg, lg, sz, vp, vp, vp]
    for name, p in (("nnhip_attn_chunk", pg), ("nnhip_attn_chunk8", p8)):
        getattr(lib, name).argtypes = [p, vp, lg, lg, sz, sz, vp, sz, vp, vp, f, vp, lg, lg, vp, vp, vp, sz, vp]
        ws = getattr(lib, name + "_workspace_bytes")
        ws.argtypes, ws.restype = [p, sz, sz, sz], sz
    lib.nnhip_draft_verify.argtypes = [vp, sz, vp, sz, i32, sz, sz, vp, vp, sz, sz, f, vp, vp, vp, vp, vp, sz, vp]
    lib.nnhip_draft_verify_workspace_bytes.argtypes = [sz, sz, sz, sz]
    lib.nnhip_draft_verify_workspace_bytes.restype = sz
    return lib


def prepare(case, seed):
    """The lengths are on the host too, as the program that hands out the pages has them."""
    return dict(case=case, x=_INPUTS[case["kind"]](case, seed), sizes=_sizes(case))


# -- one pass: the framework's calls -------------------------------------------
def _call(rc):
    if rc != 0:
        raise RuntimeError(f"the kernel library returned {rc}")


def _lib_of(st):
    if "lib" not in st:
        st["lib"] = _library()
        if st["case"]["kind"] != "verify":
            st["pg"] = _pages(st["case"], st["x"])
    return st["lib"]


def _read_back(st, c, x, n, stream):
    kv = _strides(c, n, c["heads"])
    _call(st["lib"].nnhip_kv8_read(st["pg"], x["k_back"].data_ptr(), *kv, x["v_back"].data_ptr(), *kv, n, x["seq"].data_ptr(),
                                   x["pos"].data_ptr(), stream))
    return [x["k_back"], x["v_back"]]


def _own_store(st, c, x, stream):
    lib, n = _lib_of(st), c["tokens"]
    kv, qs = _strides(c, n, c["heads"]), _strides(c, n, c["q_heads"])
    rope = c["rope"] > 0
    _call(lib.nnhip_kv8_append(st["pg"], x["k"].data_ptr(), *kv, x["v"].data_ptr(), *kv, x["q"].data_ptr(), *qs,
                               x["out"].data_ptr(), *qs, c["q_heads"], n, x["seq"].data_ptr(), x["pos"].data_ptr(),
                               x["cos"].data_ptr() if rope else None, x["sin"].data_ptr() if rope else None,
                               x["cos"].shape[0] if rope else 0, c["rope"], stream))
    return [x["out"], x["Ks"], x["Vs"]] + _read_back(st, c, x, n, stream)


def _own_read(st, c, x, stream):
    _lib_of(st)
    return _read_back(st, c, x, x["pos"].numel(), stream)


def _own_chunk(st, c, x, stream):
    lib = _lib_of(st)
    name, n, most = "nnhip_attn_chunk" + ("8" if c["bits"] == 8 else ""), sum(st["sizes"]["count"]), c["new"]
    if "ws" not in st:
        need = getattr(lib, name + "_workspace_bytes")(st["pg"], c["q_heads"], n, most)
        st["ws"] = torch.empty(max(1, need // 4), device="cuda")
    qs = _strides(c, n, c["q_heads"])
    _call(getattr(lib, name)(st["pg"], x["q"].data_ptr(), *qs, c["q_heads"], n, x["start"].data_ptr(), most, x["lens"].data_ptr(),
                             None if x["slopes"] is None else x["slopes"].data_ptr(), 1.0 / math.sqrt(c["dim"]),
                             x["out"].data_ptr(), *qs, None, None, st["ws"].data_ptr(), 4 * st["ws"].numel(), stream))
    return [x["out"]]


def _own_verify(st, c, x, stream):
    lib = _lib_of(st)
    n, b, most = sum(st["sizes"]["count"]), c["batch"], c["drafted"] + 1
    if "ws" not in st:
        need = lib.nnhip_draft_verify_workspace_bytes(n, b, most, c["vocab"])
        st["ws"] = torch.empty(max(1, need // 4), device="cuda")
        st["out"] = [torch.empty(b, device="cuda") for _ in range(2)]
    ld = c["vocab"] if c["token_major"] else n
    _call(lib.nnhip_draft_verify(x["target"].data_ptr(), ld, None if x["draft"] is None else x["draft"].data_ptr(), ld,
                                 int(c["token_major"]), c["vocab"], n, x["fed"].data_ptr(), x["start"].data_ptr(), b, most,
                                 c["temperature"], x["accept"].data_ptr(), x["pick"].data_ptr(),
                                 *[t.data_ptr() for t in st["out"]], st["ws"].data_ptr(), 4 * st["ws"].numel(), stream))
    return st["out"]


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


def _live(x):
    live = torch.nonzero(x["pos"] >= 0)[:, 0]
    return live, x["seq"][live].long(), x["pos"][live].long()


def _plain_back(c, x, live, rows):
    n = len(live)
    for back, t, s in (("k_back", "K", "Ks"), ("v_back", "V", "Vs")):
        y = x[t][rows].float().reshape(n, c["heads"], c["dim"]) * x[s][rows][..., None]
        _tokens(c, x[back])[live] = y.reshape(n, -1)
    return [x["k_back"], x["v_back"]]


def _plain_store(st, c, x):
    live, seq, pos = _live(x)
    rows = _row_index(c, x["table"], seq, pos)
    cos, sin = x["cos"][pos], x["sin"][pos]
    k, v = (_tokens(c, x[n])[live].reshape(-1, c["heads"], c["dim"]).double() for n in "kv")
    k = _rotate(c, k, cos.double(), sin.double())   # 64 bits: next to a border of two bytes
    for y, t, s in ((k, "K", "Ks"), (v, "V", "Vs")):
        scale = (y.abs().amax(2) / 127).float()
        by = torch.round(y / scale.double()[..., None]).clamp(-127, 127)
        x[t][rows] = by.to(torch.int8).reshape(len(live), -1)
        x[s][rows] = scale
    q = _tokens(c, x["q"])[live].reshape(-1, c["q_heads"], c["dim"])
    _tokens(c, x["out"])[live] = _rotate(c, q, cos, sin).reshape(len(live), -1)
    return [x["out"], x["Ks"], x["Vs"]] + _plain_back(c, x, live, rows)


def _plain_read(st, c, x):
    live, seq, pos = _live(x)
    return _plain_back(c, x, live, _row_index(c, x["table"], seq, pos))


def _cached(c, x, name, rows):
    """Keys or values of rows, (heads, n, dim) in 32 bits."""
    y = x[name][rows].float().reshape(len(rows), c["heads"], c["dim"])
    if c["bits"] == 8:
        y = y * x[name + "s"][rows][..., None]
    return y.permute(1, 0, 2).contiguous()


def _plain_chunk(st, c, x):
    kh, r, d = c["heads"], c["q_heads"] // c["heads"], c["dim"]
    starts, out = _starts(st["sizes"]["count"]), []
    for b, (new, past) in enumerate(zip(st["sizes"]["count"], st["sizes"]["past"])):
        n = new + past
        pos = torch.arange(n, device="cuda")
        rows = _row_index(c, x["table"], b, pos)
        K, V = _cached(c, x, "K", rows), _cached(c, x, "V", rows)
        q = _tokens(c, x["q"])[starts[b]:starts[b] + new].reshape(new, kh, r, d).permute(1, 2, 0, 3).reshape(kh, r * new, d)
        s = torch.matmul(q.contiguous(), K.transpose(1, 2).contiguous()).reshape(kh, r, new, n) * (1.0 / math.sqrt(d))
        own_pos = past + torch.arange(new, device="cuda")[:, None]
        if x["slopes"] is not None:
            s = s - x["slopes"].reshape(kh, r, 1, 1) * (own_pos - pos)
        s = torch.where(pos <= own_pos, s, -math.inf)
        e = torch.exp(s - s.amax(3, keepdim=True))
        total = e.sum(3, keepdim=True)
        o = torch.matmul(e.reshape(kh, r * new, n), V).reshape(kh, r, new, d) / total
        out.append(o.permute(2, 0, 1, 3).reshape(new, -1))
    out = torch.cat(out)
    return [out.t().contiguous() if c["feature_major"] else out]


def _probabilities(c, z):
    z = z.double() / c["temperature"]   # 64 bits: a random number next to a border
    e = torch.exp(z - z.amax(1, keepdim=True))
    return e / e.sum(1, keepdim=True)


def _plain_verify(st, c, x):
    v, count = c["vocab"], torch.tensor(st["sizes"]["count"], device="cuda")
    start = x["start"].long()
    target = x["target"] if c["token_major"] else x["target"].t()
    n = target.shape[0]
    row = torch.arange(n, device="cuda")
    fed = torch.zeros(n, dtype=torch.long, device="cuda")
    fed[:-1] = x["fed"][1:].long()   # the token drafted after a row
    last = start[1:] - 1
    if c["temperature"] > 0:
        p = _probabilities(c, target)
        if x["draft"] is None:
            q = torch.zeros_like(p)
            q[row, fed] = 1.0
        else:
            q = _probabilities(c, x["draft"] if c["token_major"] else x["draft"].t())
        stands = x["accept"].double() * q[row, fed] < p[row, fed]
    else:
        best = target.argmax(1)
        stands = best == fed
    stands[last] = False
    # The first row of each sequence that does not stand.
    fails = torch.where(stands, n, row)
    owner = torch.repeat_interleave(torch.arange(len(count), device="cuda"), count)
    at = torch.full((len(count),), n, device="cuda").scatter_reduce(0, owner, fails, "amin")
    accepted = (at - start[:-1]).float()
    if c["temperature"] > 0:
        left = torch.where((at == last)[:, None], p[at], (p[at] - q[at]).clamp(min=0))
        left = torch.where(left.sum(1, keepdim=True) > 0, left, p[at])
        up = torch.cumsum(left, 1)
        token = (up <= x["pick"].double()[:, None] * up[:, -1:]).sum(1).clamp(max=v - 1).float()
    else:
        token = best[at].float()
    return [accepted, token]


def run(state):
    c, x = state["case"], state["x"]
    if own:
        stream = torch.cuda.current_stream().cuda_stream
        return {"store": _own_store, "read": _own_read, "chunk": _own_chunk, "verify": _own_verify}[c["kind"]](state, c, x, stream)
    return {"store": _plain_store, "read": _plain_read, "chunk": _plain_chunk, "verify": _plain_verify}[c["kind"]](state, c, x)


# -- what a pass cannot do without -------------------------------------------
def work(case):
    c, s = case, _sizes(case)
    if c["kind"] == "store":
        n = c["tokens"] - c["pad"]
        kv = 2 * n * c["heads"]   # heads' rows: read in float32, stored as bytes and a scale, read back
        return dict(bytes=kv * (4.0 * c["dim"] + 2 * (c["dim"] + 4.0) + 4.0 * c["dim"]) + 8.0 * n * c["q_heads"] * c["dim"]
                    + 4.0 * n * (c["rope"] + 3), flops=3.0 * n * c["rope"] * (c["heads"] + c["q_heads"]) + 4.0 * kv * c["dim"])
    if c["kind"] == "read":
        kv = 2 * sum(s["len"]) * c["heads"]
        return dict(bytes=kv * (5.0 * c["dim"] + 4.0) + 12.0 * sum(s["len"]), flops=1.0 * kv * c["dim"])
    if c["kind"] == "chunk":
        rows = sum(n + p for n, p in zip(s["count"], s["past"]))
        seen = sum(n * p + n * (n + 1) // 2 for n, p in zip(s["count"], s["past"]))
        of_row = 2.0 * c["heads"] * (4.0 * c["dim"] if c["bits"] == 32 else c["dim"] + 4.0)
        return dict(bytes=rows * (of_row + 4.0 / c["page"]) + 8.0 * c["dim"] * c["q_heads"] * sum(s["count"]),
                    flops=4.0 * c["dim"] * c["q_heads"] * seen)
    n, b = sum(s["count"]), c["batch"]
    both = n + (n - b if c["draft"] else 0) if c["temperature"] > 0 else n   # the draft has no say behind its last token
    return dict(bytes=4.0 * both * c["vocab"] + 8.0 * n + 16.0 * b, flops=5.0 * both * c["vocab"])


# -- the same results in 64 bits ---------------------------------------------
def _exact_rows(c, x):
    """Each token's row of the cache, None for padding, by plain loops."""
    table = x["table"].cpu().numpy()
    rows = []
    for b, p in zip(x["seq"].long().tolist(), x["pos"].long().tolist()):
        rows.append(None if p < 0 else int(table[b, p // c["page"]]) * c["page"] + p % c["page"])
    return rows


def _exact_store(c, x):
    at = [n for n, r in enumerate(_exact_rows(c, x)) if r is not None]
    row = [r for r in _exact_rows(c, x) if r is not None]
    pos = x["pos"].long()[at]
    half = c["rope"] // 2

    def by_head(name, heads):
        t = x[name].T if c["feature_major"] else x[name]
        return t.double().reshape(c["tokens"], heads, c["dim"])[at].clone()

    def turned(z):
        if half:   # a pair as a complex number times e^(i angle)
            w = torch.complex(z[..., :half].clone(), z[..., half:2 * half].clone())
            w = w * torch.complex(x["cos"].double()[pos], x["sin"].double()[pos])[:, None, :]
            z[..., :half], z[..., half:2 * half] = w.real, w.imag
        return z

    outs = [x["out"].double()]
    (outs[0].T if c["feature_major"] else outs[0])[at] = turned(by_head("q", c["q_heads"])).reshape(len(at), -1)
    backs = []
    for y, scales, back in ((turned(by_head("k", c["heads"])), x["Ks"], x["k_back"]), (by_head("v", c["heads"]), x["Vs"], x["v_back"])):
        y = y.cpu().numpy()
        scale = (np.abs(y).max(axis=2) / 127).astype(np.float32)
        stands_for = np.rint(y / scale.astype(np.float64)[..., None]) * scale.astype(np.float64)[..., None]
        whole = scales.double()
        whole[row] = torch.from_numpy(scale).double().cuda()
        outs.append(whole)
        b = back.double()
        (b.T if c["feature_major"] else b)[at] = torch.from_numpy(stands_for).reshape(len(at), -1).cuda()
        backs.append(b)
    return outs + backs


def _exact_read(c, x):
    row = torch.tensor(_exact_rows(c, x), device="cuda")
    out = []
    for t, s in (("K", "Ks"), ("V", "Vs")):
        y = (x[t].double().reshape(-1, c["heads"], c["dim"]) * x[s].double().unsqueeze(2))[row].reshape(len(row), -1)
        out.append(y.T.contiguous() if c["feature_major"] else y)
    return out


def _exact_chunk(c, x):
    r, d = c["q_heads"] // c["heads"], c["dim"]
    q = (x["q"].T if c["feature_major"] else x["q"]).double().reshape(-1, c["heads"], r, d)
    out = torch.zeros_like(q)
    start = x["start"].long().tolist()
    for b, n in enumerate(x["lens"].long().tolist()):
        j = torch.arange(n, device="cuda")
        row = x["table"][b].long()[j // c["page"]] * c["page"] + j % c["page"]
        lo, hi = start[b], start[b + 1]
        p = n - (hi - lo) + torch.arange(hi - lo, device="cuda")
        for h in range(c["heads"]):
            K, V = (x[t].reshape(-1, c["heads"], d)[row, h].double() for t in "KV")
            if c["bits"] == 8:
                K, V = K * x["Ks"][row, h].double()[:, None], V * x["Vs"][row, h].double()[:, None]
            for i in range(r):
                s = (q[lo:hi, h, i] @ K.T.contiguous()) / math.sqrt(d)
                if x["slopes"] is not None:
                    s = s - x["slopes"].double()[h * r + i] * (p[:, None] - j)
                s = s.masked_fill(j > p[:, None], -math.inf)
                out[lo:hi, h, i] = torch.softmax(s, dim=1) @ V
    out = out.reshape(out.shape[0], -1)
    return [out.T.contiguous() if c["feature_major"] else out]


def _exact_verify(c, x):
    rows = lambda t: None if t is None else (t if c["token_major"] else t.T).cpu().numpy().astype(np.float64)  # noqa: E731
    target, draft = rows(x["target"]), rows(x["draft"])
    fed, start = x["fed"].long().tolist(), x["start"].long().tolist()
    u, w = x["accept"].double().tolist(), x["pick"].double().tolist()

    def p_of(z):
        z = z / c["temperature"]
        return np.exp(z - (z.max() + np.log(np.exp(z - z.max()).sum())))

    accepted, tokens = [], []
    for b in range(c["batch"]):
        lo, hi = start[b], start[b + 1]
        for i in range(lo, hi):
            token = fed[i + 1] if i + 1 < hi else None
            if c["temperature"] == 0:
                best = int(np.flatnonzero(target[i] == target[i].max())[0])
                if token == best:
                    continue
                tokens.append(best)
                break
            p = p_of(target[i])
            if token is None:
                left = p
            else:
                q = p_of(draft[i]) if draft is not None else (np.arange(c["vocab"]) == token).astype(np.float64)
                if u[i] * q[token] < p[token]:
                    continue
                left = np.maximum(p - q, 0)
                left = left if left.sum() > 0 else p
            up = np.cumsum(left)
            tokens.append(min(int(np.searchsorted(up, w[b] * up[-1], side="right")), c["vocab"] - 1))
            break
        accepted.append(i - lo)
    return [torch.tensor(accepted, dtype=torch.float64), torch.tensor(tokens, dtype=torch.float64)]


def exact(case, seed):
    x = _INPUTS[case["kind"]](case, seed)
    return {"store": _exact_store, "read": _exact_read, "chunk": _exact_chunk, "verify": _exact_verify}[case["kind"]](case, x)
