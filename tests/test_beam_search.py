"""The engine's paged-cache and beam-search calls and the GPT session's beam search on the CPU oracle, against plain
numpy forms and a float64 beam search over an independent forward pass."""
import ctypes

import numpy as np
import pytest

import beam_reference
import nnengine
import paged_helpers as ph
import torch_gpt

SMALL = dict(vocab_size=23, d_model=16, seq_len=14, num_heads=2, d_ff=24, num_layers=2)
VARIANTS = [dict(pos_enc="learned"), dict(pos_enc="sinusoidal", activation="gelu", norm="layernorm"), dict(pos_enc="alibi"),
            dict(pos_enc="rope")]


def params_of(cfg, seed, std=0.4):
    rng = np.random.default_rng(seed)
    return [rng.normal(0, std, s).astype(np.float32) for s in torch_gpt.param_shapes(cfg)]


def check_beams(found, params, prompt, beams, max_new, eos, cfg):
    """The totals are the reference's and each is its tokens' own (float32 logits: 1e-3 over a dozen steps of totals
    around -30); the tokens too, unless two totals that were compared lie closer than that."""
    want, gap = beam_reference.beam_search(params, prompt, beams, max_new, eos, cfg)
    import torch
    p64 = [torch.as_tensor(np.asarray(p, np.float64)) for p in params]
    assert len(found) == beams
    steps = min(max_new, cfg["seq_len"] - len(prompt) + 1)
    for (toks, score), (wt, ws, _) in zip(found, want):
        assert abs(score - ws) <= 1e-3
        assert abs(score - beam_reference.total(p64, prompt, toks, eos if len(toks) < steps else None, cfg)) <= 1e-3
    if gap > 2e-3:
        assert [t for t, _ in found] == [t for t, _, _ in want]
    return gap


@pytest.mark.parametrize("variant", VARIANTS, ids=lambda v: v["pos_enc"])
@pytest.mark.parametrize("beams,n_prompt,max_new", [(1, 3, 5), (4, 5, 6), (7, 1, 20), (3, 14, 4), (23, 2, 3), (5, 13, 9)])
def test_session_beam_search(cpu, variant, beams, n_prompt, max_new):
    cfg = dict(SMALL, **variant)
    params = params_of(cfg, 3)
    g = cpu.gpt(**cfg)
    g.set_params(params)
    prompt = np.random.default_rng(beams + n_prompt).integers(0, 23, n_prompt).tolist()
    for eos in (5, 23):
        check_beams(g.beam_search(prompt, beams, max_new, eos), params, prompt, beams, max_new, eos, cfg)


def test_long_prompt(cpu):
    """More tokens than are taken at a time: later ones share what was stored before."""
    cfg = dict(SMALL, seq_len=160, pos_enc="alibi")
    params = params_of(cfg, 4)
    g = cpu.gpt(**cfg)
    g.set_params(params)
    prompt = np.random.default_rng(1).integers(0, 23, 150).tolist()
    check_beams(g.beam_search(prompt, 4, 5, 5), params, prompt, 4, 5, 5, cfg)


def test_backward_needs_its_own_forward(cpu):
    cfg = dict(SMALL, pos_enc="learned")
    g = cpu.gpt(**cfg)
    g.set_params(params_of(cfg, 7))
    toks = np.random.default_rng(0).integers(0, 23, (15, 2))
    g.load_batch(toks[:14].astype(np.float32), toks[1:].T.reshape(-1))
    g.forward_loss()
    g.backward()
    grads = g.grads()
    g.zero_grad()
    g.forward_loss()
    g.beam_search([1, 2], 3, 2)
    with pytest.raises(nnengine.EngineError, match="forward pass"):
        g.backward()
    g.forward_loss()
    g.backward()
    assert all(np.array_equal(a, b) for a, b in zip(grads, g.grads()))


def test_one_beam_is_greedy(cpu):
    cfg = dict(SMALL, pos_enc="rope")
    g = cpu.gpt(**cfg)
    g.set_params(params_of(cfg, 5))
    assert g.beam_search([1, 2, 3], 1, 8)[0][0] == g.generate([1, 2, 3], 8)


def test_session_refusals(cpu):
    cfg = dict(SMALL, pos_enc="learned")
    g = cpu.gpt(**cfg)
    for args, msg in [(([], 2, 3), "empty prompt"), (([23], 2, 3), "out of range"), (([1] * 15, 2, 3), "longer than"),
                      (([1], 0, 3), "beams"), (([1], 257, 3), "beams"), (([1], 24, 3), "more beams"),
                      (([1], 2, -1), "max_new"), (([1], -1, 3), "beams")]:
        with pytest.raises(nnengine.EngineError, match=msg):
            g.beam_search(*args)
    assert g.beam_search([1, 2], 3, 0) == [([], 0.0)] * 3
    f = cpu._f["gpt_beam_search"]
    one = (ctypes.c_uint64 * 1)(1)
    assert f(g._g, one, 1, 1, 1, 0, None, None, None) != 0
    assert f(None, one, 1, 1, 1, 0, one, (ctypes.c_size_t * 1)(), (ctypes.c_float * 1)()) != 0
    wide = cpu.gpt(vocab_size=16, d_model=136, seq_len=8, num_heads=1, d_ff=8, num_layers=1, pos_enc="learned")
    with pytest.raises(nnengine.EngineError, match="128"):
        wide.beam_search([1], 2, 2)


# -- the calls one by one ----------------------------------------------------------
def run_ops(e, seed=0, slopes=True):
    """append, attention, selection and reordering through an engine; the inputs and every output."""
    rng = np.random.default_rng(seed)
    heads, qh, d, page, width, B, vocab = 2, 4, 8, 4, 5, 6, 50
    pages = 40
    table = rng.permutation(pages)[:B * width].reshape(B, width).astype(np.float32)
    table[1:3, :2] = table[0, :2]
    table[4, 3] = -1
    lens = np.array([17, 9, 20, 3, 16, 0], np.float32)
    x = dict(K=rng.normal(size=(pages * page, heads * d)), V=rng.normal(size=(pages * page, heads * d)), table=table,
             k=rng.normal(size=(heads * d, B)), v=rng.normal(size=(heads * d, B)), q=rng.normal(size=(qh * d, B)),
             pos=np.maximum(lens - 1, -1)[:, None], lens=lens[:, None], cos=rng.normal(size=(30, 3)),
             sin=rng.normal(size=(30, 3)), seq=np.array([0, 1, 2, 3, 4, -1])[:, None],
             shared=np.array([8, 0.0])[:, None], slopes=2.0 ** -np.arange(1, qh + 1)[:, None],
             logits=rng.normal(0, 2, (vocab, B)), scores=rng.uniform(-5, 0, (B, 1)), done=np.array([0, 0, 1, 0, 0, 0.0])[:, None],
             fresh=np.array([35, 36, 37, 38, 39, 34.0])[:, None])
    x = {n: np.asarray(a, np.float32) for n, a in x.items()}
    x["fresh"] = np.setdiff1d(np.arange(pages), table.reshape(-1))[:B].astype(np.float32)[:, None]
    t = {n: e.tensor(a) for n, a in x.items()}
    out = dict(qr=e.kv_append(t["K"], t["V"], t["table"], t["k"], t["v"], t["pos"], page, heads, q=t["q"], cos=t["cos"],
                              sin=t["sin"], seq=t["seq"]))
    out["O"] = e.attn_paged(t["K"], t["V"], t["table"], out["qr"], t["lens"], 0.3, page, heads, shared=t["shared"], group=3,
                            slopes=t["slopes"] if slopes else None)
    out["score"], out["beam"], out["token"] = e.beam_select(t["logits"], t["scores"], 4, done=t["done"], groups=2, eos=7)
    parent = e.tensor(np.array([[0.0], [0], [2], [4], [3], [9]]))
    out["table2"], out["lens2"] = e.kv_reorder([(t["K"], t["V"])], t["table"], parent, t["lens"], t["fresh"], page, heads)
    out["K"], out["V"] = t["K"], t["V"]
    return x, {n: a.numpy() for n, a in out.items()}


def test_calls_against_numpy(cpu):
    x, got = run_ops(cpu)
    heads, qh, d, page, pages, B, h = 2, 4, 8, 4, 40, 6, 3
    K, V, qr = x["K"].astype(np.float64), x["V"].astype(np.float64), x["q"].astype(np.float64).copy()

    def turned(a, p):
        a = a.astype(np.float64).reshape(-1, d).copy()
        lo, hi = a[:, :h].copy(), a[:, h:2 * h].copy()
        a[:, :h], a[:, h:2 * h] = lo * x["cos"][p] - hi * x["sin"][p], hi * x["cos"][p] + lo * x["sin"][p]
        return a.reshape(-1)

    for n in range(B):
        b, p = ph.index_of(x["seq"][n, 0], B), ph.index_of(x["pos"][n, 0], 30)
        r = None if b is None or p is None else ph.row_of(x["table"], b, p, page, pages)
        if r is not None:
            K[r], V[r], qr[:, n] = turned(x["k"][:, n], p), x["v"][:, n], turned(x["q"][:, n], p)
    assert np.abs(got["qr"] - qr).max() <= 1e-5
    Kh, Vh = K.reshape(-1, heads, d), V.reshape(-1, heads, d)
    wO, _, _, _ = ph.attend(qr.T.reshape(B, qh, d), Kh, Vh, x["table"], page, pages, heads, x["lens"][:, 0], 0.3,
                            x["slopes"][:, 0])
    assert np.abs(got["O"].T.reshape(B, qh, d) - wO).max() <= 1e-5
    sel = ph.select(x["logits"].T.reshape(2, 3, -1), x["scores"].reshape(2, 3), x["done"].reshape(2, 3), 4, 7)
    assert np.array_equal(got["beam"], sel[1]) and np.array_equal(got["token"], sel[2])
    assert np.abs(got["score"] - sel[0]).max() <= 1e-5
    t2, l2, (K2, V2) = ph.reorder([K, V], x["table"], page, pages, [0, 0, 2, 4, 3, 9], x["lens"][:, 0], x["fresh"][:, 0], 5)
    assert np.array_equal(got["table2"], t2) and np.array_equal(got["lens2"][:, 0], l2)
    assert np.abs(got["K"] - K2).max() <= 1e-5 and np.abs(got["V"] - V2).max() <= 1e-5


def refusals(e):
    """(call, message) of shapes that do not fit."""
    T = e.create_tensor
    K, V, table, x, col = T(8, 6), T(8, 6), T(3, 2), T(6, 3), T(3, 1)
    for t in (K, V, table, x, col):
        e.zero(t)
    return [
        (lambda: e.kv_append(K, V, table, x, x, col, 3, 2), "cache shapes"),
        (lambda: e.kv_append(K, K, table, x, x, col, 2, 2), "one tensor"),
        (lambda: e.kv_append(K, V, table, x, x, col, 2, 4), "cache shapes"),
        (lambda: e.kv_append(K, V, table, x, x, col, 0, 2), "cache shapes"),
        (lambda: e.kv_append(K, V, table, x, T(6, 2), col, 2, 2), "k, v"),
        (lambda: e.kv_append(K, V, table, x, x, T(2, 1), 2, 2), "one position"),
        (lambda: e.kv_append(K, V, table, x, x, col, 2, 2, seq=T(2, 1)), "one position"),
        (lambda: e.kv_append(K, V, table, x, x, col, 2, 2, q=T(7, 3)), "q shape"),
        (lambda: e.kv_append(K, V, table, x, x, col, 2, 2, cos=T(4, 2), sin=T(4, 2)), "cos, sin"),
        (lambda: e.kv_append(K, V, table, x, x, col, 2, 2, cos=T(4, 1), sin=T(5, 1)), "cos, sin"),
        (lambda: e.kv_append(K, V, table, x, x, col, 2, 2, cos=T(4, 1)), "go together"),
        (lambda: e.attn_paged(K, V, table, T(6, 2), col, 1.0, 2, 2), "q shape"),
        (lambda: e.attn_paged(K, V, table, T(9, 3), col, 1.0, 2, 2), "q shape"),
        (lambda: e.attn_paged(K, V, table, x, T(2, 1), 1.0, 2, 2), "one length"),
        (lambda: e.attn_paged(K, V, table, x, col, 1.0, 2, 2, group=2), "groups"),
        (lambda: e.attn_paged(K, V, table, x, col, 1.0, 2, 2, group=0), "groups"),
        (lambda: e.attn_paged(K, V, table, x, col, 1.0, 2, 2, shared=col, group=3), "groups"),
        (lambda: e.attn_paged(K, V, table, x, col, 1.0, 2, 2, slopes=col), "one slope"),
        (lambda: e.beam_select(T(10, 3), T(2, 1), 2), "one score"),
        (lambda: e.beam_select(T(10, 3), col, 2, groups=2), "groups"),
        (lambda: e.beam_select(T(10, 3), col, 0), "take"),
        (lambda: e.beam_select(T(10, 3), col, 31), "take"),
        (lambda: e.beam_select(T(10, 3), col, 2, done=col, eos=10), "eos"),
        (lambda: e.beam_select(T(10, 3), col, 2, done=T(2, 1)), "done"),
        (lambda: e.kv_reorder([], table, col, col), "no layers"),
        (lambda: e.kv_reorder([(K, V)], table, col, T(2, 1), None, 2, 2), "one length"),
        (lambda: e.kv_reorder([(K, V)], table, col, col, T(2, 1), 2, 2), "parent and fresh"),
        (lambda: e.kv_reorder([(K, V), (T(10, 6), V)], table, col, col, None, 2, 2), "cache shapes"),
    ]


def test_refusals(cpu):
    for call, msg in refusals(cpu):
        with pytest.raises(nnengine.EngineError, match=msg):
            call()


def test_refused_search_leaves_the_forward_pass(cpu):
    """A search that is refused, or asked for no token, has run no layer: the backward pass still has its inputs."""
    cfg = dict(SMALL, pos_enc="learned")
    g = cpu.gpt(**cfg)
    g.set_params(params_of(cfg, 7))
    toks = np.random.default_rng(0).integers(0, 23, (15, 2))
    g.load_batch(toks[:14].astype(np.float32), toks[1:].T.reshape(-1))
    g.forward_loss()
    g.backward()
    grads = g.grads()
    for args in ([1] * 15, 2, 3), ([1], 257, 3), ([1], 24, 3), ([23], 2, 3), ([], 2, 3):
        g.zero_grad()
        g.forward_loss()
        with pytest.raises(nnengine.EngineError):
            g.beam_search(*args)
        g.backward()
        assert all(np.array_equal(a, b) for a, b in zip(grads, g.grads()))
    g.zero_grad()
    g.forward_loss()
    f, one, n, s = cpu._f["gpt_beam_search"], (ctypes.c_uint64 * 1)(1), (ctypes.c_size_t * 3)(), (ctypes.c_float * 3)()
    assert f(g._g, one, 1, 0, 3, 0, one, n, s) != 0
    assert g.beam_search([1, 2], 3, 0) == [([], 0.0)] * 3
    g.backward()
    assert all(np.array_equal(a, b) for a, b in zip(grads, g.grads()))
    wide = cpu.gpt(vocab_size=23, d_model=136, seq_len=14, num_heads=1, d_ff=8, num_layers=1, pos_enc="learned")
    wide.load_batch(toks[:14].astype(np.float32), toks[1:].T.reshape(-1))
    wide.forward_loss()
    with pytest.raises(nnengine.EngineError, match="128"):
        wide.beam_search([1], 2, 2)
    wide.backward()


def orphan_first(e, beams):
    """The first sequences of a group continue no one (a table row of -1, length 0); the others share a prefix."""
    rng = np.random.default_rng(11)
    heads, d, page, width, pages, n = 2, 32, 4, 12, 120, 37
    x = dict(K=rng.normal(size=(pages * page, heads * d)), V=rng.normal(size=(pages * page, heads * d)),
             q=rng.normal(size=(heads * d, beams)), table=np.full((1, width), -1.0), lens=np.array([[n]]))
    x["table"][0, :n // page + 1] = rng.permutation(30)[:n // page + 1]
    parent = np.zeros((beams, 1))
    parent[:max(1, beams - 5)] = -1
    x = {k: np.asarray(a, np.float32) for k, a in x.items()}
    t = {k: e.tensor(a) for k, a in x.items()}
    fresh = e.tensor(40.0 + np.arange(beams)[:, None])
    table, lens = e.kv_reorder([(t["K"], t["V"])], t["table"], e.tensor(parent), t["lens"], fresh, page, heads)
    got = e.attn_paged(t["K"], t["V"], table, t["q"], lens, 0.2, page, heads, shared=e.tensor(np.array([[n // page * page]])),
                       group=beams).numpy()
    K, V = (t[k].numpy().reshape(-1, heads, d) for k in "KV")
    want, _, _, tol = ph.attend(x["q"].T.reshape(beams, heads, d), K, V, table.numpy(), page, pages, heads, lens.numpy()[:, 0],
                                np.float32(0.2))
    assert np.all(lens.numpy()[parent[:, 0] < 0] == 0) and np.all(np.abs(want[parent[:, 0] == 0]).sum(axis=(1, 2)) > 0)
    assert np.all(np.abs(got.T.reshape(beams, heads, d) - want) <= tol)


@pytest.mark.parametrize("beams", [2, 6, 70])
def test_group_whose_first_sequence_has_no_parent(cpu, beams):
    orphan_first(cpu, beams)


def test_any_number_of_new_tokens(cpu):
    """More tokens than the context has room for are what fits, however many are asked for."""
    cfg = dict(SMALL, pos_enc="rope")
    g = cpu.gpt(**cfg)
    g.set_params(params_of(cfg, 5))
    want = g.beam_search([1, 2, 3], 4, 12, 5)
    for n in (13, 14, 10 ** 6, 10 ** 15, 2 ** 64 - 1):
        assert g.beam_search([1, 2, 3], 4, n, 5) == want


def through_views(e):
    """Caches, tokens and tables that are slices of other tensors, or are sliced before they are written: a slice is a
    copy, whatever is written afterwards on either side."""
    rng = np.random.default_rng(21)
    heads, d, page, pages, n = 2, 4, 2, 8, 8
    both = e.tensor(rng.normal(size=(2 * pages * page, heads * d)).astype(np.float32))
    tables = e.tensor(np.arange(4 * 4, dtype=np.float32).reshape(4, 4) % pages)
    out = {}
    K, V = e.slice_rows(both, 0, pages * page), e.slice_rows(both, pages * page, pages * page)
    table = e.slice_rows(tables, 1, 2)
    k, v = e.slice_rows(K, 0, heads * d), e.slice_rows(both, 3, heads * d)     # (heads * d, 8 tokens)
    before = e.slice_rows(K, 2, 9)
    seq = e.tensor((np.arange(n) % 2).astype(np.float32)[:, None])
    pos = e.tensor((np.arange(n) // 2).astype(np.float32)[:, None])
    cos, sin = (e.tensor(rng.normal(size=(8, 2)).astype(np.float32)) for _ in range(2))
    out["q"] = e.kv_append(K, V, table, k, v, pos, page, heads, q=k, cos=cos, sin=sin, seq=seq)
    after = e.slice_rows(K, 2, 9)
    lens = e.tensor(np.array([[3.0], [4]]))
    q2 = e.slice_rows(both, 5, 2)                                               # (2, 8): as (heads * d, batch) below
    out["O"] = e.attn_paged(K, V, table, e.transpose(q2), lens, 0.5, page, heads)
    out["table2"], out["lens2"] = e.kv_reorder([(K, V)], table, e.tensor(np.array([[1.0], [0]])), lens,
                                               e.tensor(np.array([[3.0], [6]])), page, heads)
    out.update(K=K, V=V, k=k, v=v, before=before, after=after, both=both, tables=tables)
    return {n: t.numpy() for n, t in out.items()}


def test_slices_are_copies(cpu):
    got = through_views(cpu)
    rng = np.random.default_rng(21)
    both = rng.normal(size=(32, 8)).astype(np.float32)
    assert np.array_equal(got["both"], both) and np.array_equal(got["before"], both[2:11])
    assert np.array_equal(got["k"], both[:8]) and np.array_equal(got["v"], both[3:11])
    assert not np.array_equal(got["after"], both[2:11])
