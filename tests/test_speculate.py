"""The engine's calls on chunks of new tokens, 8-bit caches and drafted tokens, and the GPT session's speculative decoding,
on the CPU oracle, against plain numpy forms and a float64 forward pass."""
import ctypes

import numpy as np
import pytest

import chunk_helpers as ch
import draft_reference
import nnengine

SMALL = dict(vocab_size=23, d_model=16, seq_len=30, num_heads=2, d_ff=24, num_layers=2)
VARIANTS = [dict(pos_enc="learned"), dict(pos_enc="sinusoidal", activation="gelu", norm="layernorm"), dict(pos_enc="alibi"),
            dict(pos_enc="rope")]
# Float32 logits of two layers of such sizes are off by less than 1e-3. A value that float32 sums put on the other side of a
# rounding moves a byte by one, so a value by the scale (at most 1/127 of its head's largest): a tenth covers that on its way
# through the second layer.
GAP = {32: 2e-3, 8: 0.1}


def params_of(cfg, seed, std=0.4):
    import torch_gpt
    rng = np.random.default_rng(seed)
    return [rng.normal(0, std, s).astype(np.float32) for s in torch_gpt.param_shapes(cfg)]


def session(e, cfg, seed, std=0.4):
    g = e.gpt(**cfg)
    p = params_of(cfg, seed, std)
    g.set_params(p)
    return g, p


def draft_of(e, cfg, seed=9):
    """A smaller model of the same vocabulary."""
    c = dict(cfg, d_model=8, num_heads=1, d_ff=12, num_layers=1)
    return session(e, c, seed)


def greedy_run(e, variant, bits, draft_len, max_new=12, eos=5):
    """Ragged prompts, a strange draft and one that agrees: the same sequences, each the definition's."""
    cfg = dict(SMALL, **variant)
    g, params = session(e, cfg, 3)
    d, _ = draft_of(e, cfg)
    rng = np.random.default_rng(draft_len + bits)
    prompts = [rng.integers(0, 23, n).tolist() for n in (4, 1, 30, 25, 9)]
    found, stats = g.speculate(d, prompts, max_new, draft_len, eos=eos, cache_bits=bits)
    clear = 0
    for f, p in zip(found, prompts):
        clear += draft_reference.check_greedy(f, params, p, max_new, eos, cfg, bits, GAP[bits])
    assert clear > 0 and stats["accepted"] <= stats["drafted"] and stats["passes"] <= max_new
    same, st = g.speculate(g, prompts, max_new, draft_len, eos=eos, cache_bits=bits)
    for f, p in zip(same, prompts):
        draft_reference.check_greedy(f, params, p, max_new, eos, cfg, bits, GAP[bits])
    return found, stats, same, st


@pytest.mark.parametrize("variant", VARIANTS, ids=lambda v: v["pos_enc"])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("draft_len", [1, 4, 11])
def test_greedy(cpu, variant, bits, draft_len):
    found, _, same, st = greedy_run(cpu, variant, bits, draft_len)
    assert found == same                     # the oracle's rounding is one and the same for any chunks
    assert st["accepted"] >= st["drafted"] - draft_len * 5   # all but what lies behind eos, of five sequences


def test_equals_generate(cpu):
    cfg = dict(SMALL, pos_enc="rope")
    g, _ = session(cpu, cfg, 5)
    d, _ = draft_of(cpu, cfg)
    for n, k in ((3, 1), (7, 3), (1, 8)):
        prompt = np.random.default_rng(n).integers(0, 23, n).tolist()
        assert g.speculate(d, [prompt], 9, k)[0][0] == g.generate(prompt, 9)
    assert g.speculate(d, [[1, 2]], 9, 3)[0] == g.speculate(d, [[1, 2], [4] * 8], 9, 5)[0][:1]


def distribution(e, bits, n=1024, rounds=4):
    """Frequencies of the first two tokens against the model's probabilities: 5 standard deviations, and 4e-3 for what the
    8-bit caches and float32 change."""
    cfg = dict(vocab_size=5, d_model=8, seq_len=12, num_heads=2, d_ff=12, num_layers=1, pos_enc="rope")
    g, params = session(e, cfg, 2, 0.5)
    d, _ = session(e, dict(cfg, d_model=4, num_heads=1), 8, 0.7)
    prompt, T, count = [1, 4, 2], 1.3, np.zeros((5, 5))
    stats = dict(drafted=0, accepted=0)
    for seed in range(rounds):
        found, st = g.speculate(d, [prompt] * n, 2, 3, temperature=T, seed=seed, cache_bits=bits)
        for f in found:
            count[f[0], f[1]] += 1
        stats = {k: stats[k] + st[k] for k in stats}
    N = n * rounds
    p1 = ch.softmax64(draft_reference.logits(params, prompt, cfg, bits)[-1], T)
    want = np.stack([p1[v] * ch.softmax64(draft_reference.logits(params, prompt + [v], cfg, bits)[-1], T) for v in range(5)])
    assert 0 < stats["accepted"] < stats["drafted"]
    assert np.all(np.abs(count / N - want) <= 5 * np.sqrt(want * (1 - want) / N) + 4e-3)


@pytest.mark.parametrize("bits", [32, 8])
def test_distribution(cpu, bits):
    distribution(cpu, bits)


def test_seeds(cpu):
    cfg = dict(SMALL, pos_enc="alibi")
    g, _ = session(cpu, cfg, 3)
    d, _ = draft_of(cpu, cfg)
    run = lambda s: g.speculate(d, [[1, 2, 3]] * 3, 12, 3, temperature=2.0, seed=s)[0]
    assert run(1) == run(1) and run(1) != run(2) and len({tuple(x) for x in run(1)}) == 3


def test_limits(cpu):
    """Context full, more tokens than fit, no tokens, one token."""
    cfg = dict(SMALL, pos_enc="learned")
    g, _ = session(cpu, cfg, 3)
    d, _ = draft_of(cpu, cfg)
    prompts = [[1] * 30, [2] * 29, [3]]
    found, _ = g.speculate(d, prompts, 10 ** 6, 7)
    assert [len(f) for f in found] == [1, 2, 30]
    none, st = g.speculate(d, prompts, 0, 7)
    assert none == [[], [], []] and st == dict(passes=0, drafted=0, accepted=0)
    one, st = g.speculate(d, prompts, 1, 7)
    assert one == [f[:1] for f in found] and st == dict(passes=1, drafted=0, accepted=0)


def test_prompt_of_several_chunks(cpu):
    cfg = dict(SMALL, seq_len=1400, pos_enc="alibi", num_layers=1)
    g, params = session(cpu, cfg, 4)
    d, _ = draft_of(cpu, cfg)
    prompt = np.random.default_rng(1).integers(0, 23, 1100).tolist()
    found, _ = g.speculate(d, [prompt, prompt[:3]], 3, 2, cache_bits=8)
    for f, p in zip(found, (prompt, prompt[:3])):
        draft_reference.check_greedy(f, params, p, 3, -1, cfg, 8, GAP[8])


def session_refusals(e):
    cfg = dict(SMALL, pos_enc="learned")
    g, _ = session(e, cfg, 1)
    d, _ = draft_of(e, cfg)
    other, _ = session(e, dict(cfg, vocab_size=24), 1)
    short, _ = session(e, dict(cfg, seq_len=10), 1)
    wide = e.gpt(vocab_size=23, d_model=136, seq_len=30, num_heads=1, d_ff=8, num_layers=1, pos_enc="learned")
    toks = np.random.default_rng(0).integers(0, 23, (31, 2))
    g.load_batch(toks[:30].astype(np.float32), toks[1:].T.reshape(-1))
    for args, kw, msg in [((d, [[]], 3), {}, "empty prompt"), ((d, [[1], [23]], 3), {}, "out of range"),
                          ((d, [[1] * 31], 3), {}, "longer than"), ((d, [[1]] * 1025, 3), {}, "1024 prompts"),
                          ((d, [], 3), {}, "no prompts"), ((d, [[1]], -1), {}, "negative"), ((d, [[1]], 3, 0), {}, "drafted"),
                          ((d, [[1]], 3, 1024), {}, "drafted"), ((d, [[1]], 3, 2, -1.0), {}, "temperature"),
                          ((d, [[1]], 3, 2, float("nan")), {}, "temperature"), ((d, [[1]], 3, 2, float("inf")), {}, "temperature"),
                          ((d, [[1]], 3), dict(cache_bits=16), "bits"), ((other, [[1]], 3), {}, "vocabulary"),
                          ((short, [[1] * 9], 3), {}, "shorter"), ((wide, [[1]], 3), {}, "128")]:
        g.forward_loss()
        with pytest.raises(nnengine.EngineError, match=msg):
            g.speculate(*args, **kw)
        g.backward()                                     # a refused call has run no layer
    with pytest.raises(nnengine.EngineError, match="128"):
        wide.speculate(d, [[1]], 3)
    assert len(g.speculate(short, [[1] * 9], 2)[0][0]) == 2   # ten positions are enough for these
    f = e._f["gpt_speculate"]
    one, n = (ctypes.c_uint64 * 4)(1), (ctypes.c_size_t * 1)(1)
    for a in ((None, d._g, one, n, one, n), (g._g, None, one, n, one, n), (g._g, d._g, None, n, one, n),
              (g._g, d._g, one, None, one, n), (g._g, d._g, one, n, None, n), (g._g, d._g, one, n, one, None)):
        assert f(a[0], a[1], a[2], a[3], 1, 1, 1, 0.0, 99, 0, 32, a[4], a[5], None) != 0
    assert f(g._g, d._g, one, n, 0, 1, 1, 0.0, 99, 0, 32, one, n, None) != 0
    assert f(g._g, d._g, one, n, 1, 1, 1, 0.0, 99, 0, 32, one, n, None) == 0


def test_session_refusals(cpu):
    session_refusals(cpu)


def test_sessions_of_two_engines(cpu):
    from conftest import oracle_engine
    cfg = dict(SMALL, pos_enc="learned")
    g, _ = session(cpu, cfg, 1)
    d, _ = session(oracle_engine(), cfg, 1)
    with pytest.raises(nnengine.EngineError, match="another engine"):
        g.speculate(d, [[1]], 3)


def backward_needs_its_own_forward(e):
    cfg = dict(SMALL, pos_enc="rope")
    (g, _), (d, _) = session(e, cfg, 7), session(e, cfg, 8)
    toks = np.random.default_rng(0).integers(0, 23, (31, 2))
    for s in (g, d):
        s.load_batch(toks[:30].astype(np.float32), toks[1:].T.reshape(-1))
        s.forward_loss()
        s.backward()
    grads = [s.grads() for s in (g, d)]
    for s in (g, d):
        s.zero_grad()
        s.forward_loss()
    g.speculate(d, [[1, 2]], 0)
    for s, want in zip((g, d), grads):
        s.backward()
        assert all(np.array_equal(a, b) for a, b in zip(want, s.grads()))
        s.zero_grad()
        s.forward_loss()
    g.speculate(d, [[1, 2]], 5)
    for s, want in zip((g, d), grads):
        with pytest.raises(nnengine.EngineError, match="forward pass"):
            s.backward()
        s.forward_loss()
        s.backward()
        assert all(np.array_equal(a, b) for a, b in zip(want, s.grads()))


def test_backward_needs_its_own_forward(cpu):
    backward_needs_its_own_forward(cpu)


# -- the calls one by one ----------------------------------------------------------
def run_ops(e, seed=0):
    """Both kinds of cache written, read back and attended to, and drafted tokens verified; inputs and outputs."""
    rng = np.random.default_rng(seed)
    heads, qh, d, page, width, B, N, vocab = 2, 4, 12, 4, 5, 4, 9, 50
    pages = 24
    table = rng.permutation(pages)[:B * width].reshape(B, width).astype(np.float32)
    table[2, 1] = -1
    x = dict(K=rng.normal(size=(pages * page, heads * d)), V=rng.normal(size=(pages * page, heads * d)), table=table,
             k=rng.normal(size=(heads * d, N)), v=rng.normal(size=(heads * d, N)), q=rng.normal(size=(qh * d, N)),
             seq=np.array([0, 0, 0, 1, 2, 2, 2, 2, -1])[:, None], pos=np.array([9, 10, 11, 0, 5, 6, 7, 8, 3])[:, None],
             start=np.array([0, 3, 4, 8, 8])[:, None], lens=np.array([12, 1, 9, 6])[:, None],
             cos=rng.normal(size=(14, 4)), sin=rng.normal(size=(14, 4)), slopes=2.0 ** -np.arange(1, qh + 1)[:, None],
             target=rng.normal(0, 2, (vocab, N)), draft=rng.normal(0, 2, (vocab, N)),
             fed=rng.integers(0, vocab, (N, 1)), accept=rng.random((N, 1)), pick=rng.random((B, 1)))
    x = {n: np.asarray(a, np.float32) for n, a in x.items()}
    x["fed"][1:3, 0] = [x["target"][:, 0].argmax(), x["target"][:, 1].argmax()]
    t = {n: e.tensor(a) for n, a in x.items()}
    out = {}
    c8 = e.kv8_cache(pages, page, heads, d)
    rope = dict(q=t["q"], cos=t["cos"], sin=t["sin"], seq=t["seq"])
    out["q8"] = e.kv8_append(c8, t["table"], t["k"], t["v"], t["pos"], page, heads, d, **rope)
    out["k8"], out["v8"] = e.kv8_read(c8, t["table"], t["pos"], page, heads, d, seq=t["seq"])
    out["O8"] = e.attn_chunk8(c8, t["table"], out["q8"], t["start"], t["lens"], 4, 0.3, page, heads, d, slopes=t["slopes"])
    out["q32"] = e.kv_append(t["K"], t["V"], t["table"], t["k"], t["v"], t["pos"], page, heads, **rope)
    out["O"] = e.attn_chunk(t["K"], t["V"], t["table"], out["q32"], t["start"], t["lens"], 3, 0.3, page, heads)
    for T in (0.0, 0.7):
        for with_draft in (True, False):
            for major in (False, True):
                tt, dd = (e.transpose(t[n]) if major else t[n] for n in ("target", "draft"))
                random = dict(accept=t["accept"], pick=t["pick"]) if T else {}
                a, k = e.draft_verify(tt, t["fed"], t["start"], 3, T, draft=dd if with_draft else None, token_major=major, **random)
                out[f"a{T}{with_draft}{major}"], out[f"t{T}{with_draft}{major}"] = a, k
    out.update(K=t["K"], V=t["V"], K8=c8[0], V8=c8[1], Ks=c8[2], Vs=c8[3])
    return x, {n: a.numpy() for n, a in out.items()}


def check_ops(x, got):
    heads, qh, d, page, width, pages, B, N = 2, 4, 12, 4, 5, 24, 4, 9
    K8, V8 = (np.zeros((pages * page, heads, d), np.int8) for _ in range(2))
    Ks, Vs = (np.zeros((pages * page, heads), np.float32) for _ in range(2))
    K, V = x["K"].astype(np.float64).reshape(-1, heads, d), x["V"].astype(np.float64).reshape(-1, heads, d)
    qr = x["q"].astype(np.float64).T.reshape(N, qh, d).copy()
    k8, v8 = np.zeros((N, heads, d)), np.zeros((N, heads, d))
    for n in range(N):
        r, p = ch.place(x["table"], B, page, pages, x["seq"][:, 0], x["pos"][:, 0], 14, n)
        if r is None:
            continue
        k = ch.turned(x["k"][:, n].reshape(heads, d), x["cos"][p], x["sin"][p], 8)
        v = x["v"][:, n].reshape(heads, d).astype(np.float64)
        qr[n] = ch.turned(x["q"][:, n].reshape(qh, d), x["cos"][p], x["sin"][p], 8)
        (K8[r], Ks[r]), (V8[r], Vs[r]) = ch.quantise(k), ch.quantise(v)
        K[r], V[r] = k, v
        k8[n], v8[n] = K8[r] * Ks[r][:, None], V8[r] * Vs[r][:, None]
    bytes_of = lambda a: a.view(np.int8).reshape(pages * page, heads, d)
    assert np.array_equal(bytes_of(got["K8"]), K8) and np.array_equal(bytes_of(got["V8"]), V8)
    assert np.array_equal(got["Ks"], Ks) and np.array_equal(got["Vs"], Vs)
    U = 2.0 ** -24
    for n, w in (("k8", k8), ("v8", v8)):
        assert np.all(np.abs(got[n].T.reshape(N, heads, d) - w) <= U * np.abs(w))
    for n in ("q8", "q32"):   # a product, a fused sum: three roundings of values up to two products' sizes
        assert np.abs(got[n].T.reshape(N, qh, d) - qr).max() <= 4 * U * 2 * np.abs(x["q"]).max() * np.abs(x["cos"]).max() + 1e-5
    assert np.abs(got["K"].reshape(K.shape) - K).max() <= 1e-5 and np.array_equal(got["V"].reshape(V.shape), V.astype(np.float32))
    f = [x[n][:, 0] for n in ("start", "lens")]
    for n, q, kv, most, slopes in (("O8", "q8", (K8 * Ks[..., None].astype(np.float64), V8 * Vs[..., None].astype(np.float64)), 4, x["slopes"][:, 0]),
                                   ("O", "q32", (got["K"].astype(np.float64).reshape(K.shape), V), 3, None)):
        w, _, _, tol, _, has = ch.attend(got[q].T.reshape(N, qh, d), *kv, x["table"], page, pages, heads, f[0], most, f[1],
                                         np.float32(0.3), slopes)
        g = got[n].T.reshape(N, qh, d)
        assert np.all(g[~has] == 0) and np.all(np.abs(g - w) <= np.maximum(tol, U))
    for T in (0.0, 0.7):
        for with_draft in (True, False):
            a, t, near = ch.verify(x["target"].T, x["draft"].T if with_draft else None, x["fed"][:, 0], f[0], 3, np.float32(T),
                                   x["accept"][:, 0], x["pick"][:, 0])
            assert near > 1e-9
            for major in (False, True):
                assert np.array_equal(got[f"a{T}{with_draft}{major}"][:, 0], a)
                assert np.array_equal(got[f"t{T}{with_draft}{major}"][:, 0], t)


@pytest.mark.parametrize("seed", [0, 1, 2])
def test_calls_against_numpy(cpu, seed):
    check_ops(*run_ops(cpu, seed))


def verified_distribution(e):
    """Over a grid of random numbers the drafted token and what replaces it follow the target: of M numbers a cut falls into
    one of M steps, twice, so each frequency is off by 2 / M at most."""
    V, M = 5, 48
    rng = np.random.default_rng(4)
    zt, zd = rng.normal(0, 1.5, V).astype(np.float32), rng.normal(0, 1.5, V).astype(np.float32)
    T = np.float32(0.8)
    p, q = ch.softmax64(zt, T), ch.softmax64(zd, T)
    g = (np.arange(M) + 0.5) / M
    x, u, w = (a.reshape(-1) for a in np.meshgrid(np.arange(V), g, g, indexing="ij"))
    n = x.size
    fed = np.zeros((2 * n, 1))
    fed[1::2, 0] = x
    accept = np.zeros((2 * n, 1))
    accept[::2, 0] = u
    a, t = e.draft_verify(e.tensor(np.repeat(zt[:, None], 2 * n, axis=1)), e.tensor(fed), e.tensor(np.arange(n + 1.0)[:, None] * 2),
                          2, float(T), draft=e.tensor(np.repeat(zd[:, None], 2 * n, axis=1)), accept=e.tensor(accept),
                          pick=e.tensor(w[:, None]))
    a, t = a.numpy()[:, 0], t.numpy()[:, 0].astype(int)
    out = np.where(a == 1, x, t)
    freq = np.zeros(V)
    np.add.at(freq, out, q[x] / (M * M))
    assert np.all(np.abs(freq - p) <= 2 / M)


def test_verified_tokens_follow_the_target(cpu):
    verified_distribution(cpu)


def refusals(e):
    """(call, message) of shapes that do not fit."""
    T = e.create_tensor
    K, V, table, x, col, st = T(8, 6), T(8, 6), T(3, 2), T(6, 3), T(3, 1), T(4, 1)
    c8 = e.kv8_cache(4, 2, 2, 3)
    for t in (K, V, table, x, col, st):
        e.zero(t)
    chunk = lambda q=x, start=st, lens=col, most=2, page=2, heads=2, **k: e.attn_chunk(K, V, table, q, start, lens, most, 1.0, page, heads, **k)
    chunk8 = lambda c=c8, q=x, start=st, lens=col, most=2, page=2, heads=2, dim=3, **k: e.attn_chunk8(c, table, q, start, lens, most, 1.0, page, heads, dim, **k)
    append = lambda c=c8, k=x, v=x, pos=col, page=2, heads=2, dim=3, **kw: e.kv8_append(c, table, k, v, pos, page, heads, dim, **kw)
    read = lambda c=c8, pos=col, page=2, heads=2, dim=3, **kw: e.kv8_read(c, table, pos, page, heads, dim, **kw)
    z = T(10, 4)
    fed, one = T(4, 1), T(3, 1)
    verify = lambda t=z, f=fed, s=st, most=2, temp=0.0, **kw: e.draft_verify(t, f, s, most, temp, **kw)
    wide = e.kv8_cache(4, 2, 1, 260)
    wide_chunk = e.kv8_cache(4, 2, 1, 132)
    return [
        (lambda: chunk(page=3), "cache shapes"), (lambda: chunk(heads=4), "cache shapes"), (lambda: chunk(q=T(7, 3)), "q shape"),
        (lambda: chunk(q=T(9, 3)), "q shape"), (lambda: chunk(start=col), "one start"), (lambda: chunk(lens=T(2, 1)), "one length"),
        (lambda: chunk(most=0), "most"), (lambda: chunk(most=4), "most"), (lambda: chunk(slopes=col), "one slope"),
        (lambda: chunk8(page=3), "cache shapes"), (lambda: chunk8(heads=3), "cache shapes"), (lambda: chunk8(dim=5), "cache shapes"),
        (lambda: chunk8(dim=0), "cache shapes"), (lambda: chunk8(q=T(7, 3)), "q shape"), (lambda: chunk8(start=col), "one start"),
        (lambda: chunk8(lens=T(2, 1)), "one length"), (lambda: chunk8(most=0), "most"), (lambda: chunk8(slopes=col), "one slope"),
        (lambda: chunk8(c=wide_chunk, q=T(132, 3), heads=1, dim=132), "cache shapes"),
        (lambda: chunk8(c=(c8[0], c8[1], c8[2], T(8, 1))), "cache shapes"),
        (lambda: append(k=T(5, 3)), "k, v"), (lambda: append(v=T(6, 2)), "k, v"), (lambda: append(pos=T(2, 1)), "one position"),
        (lambda: append(seq=T(2, 1)), "one position"), (lambda: append(q=T(7, 3)), "q shape"),
        (lambda: append(cos=T(4, 2), sin=T(4, 2)), "cos, sin"), (lambda: append(cos=T(4, 1)), "go together"),
        (lambda: append(c=(c8[0], c8[0], c8[2], c8[3])), "one tensor"), (lambda: append(c=(c8[0], c8[1], c8[2], c8[2])), "one tensor"),
        (lambda: append(c=(c8[0], T(8, 4), c8[2], c8[3])), "cache shapes"), (lambda: append(page=0), "cache shapes"),
        (lambda: append(c=wide, k=T(260, 3), v=T(260, 3), heads=1, dim=260), "cache shapes"),
        (lambda: read(page=3), "cache shapes"), (lambda: read(seq=T(2, 1)), "one sequence"), (lambda: read(pos=T(0, 1)), "no tokens"),
        (lambda: verify(f=T(5, 1)), "one token"), (lambda: verify(s=T(1, 1)), "one start"), (lambda: verify(most=0), "most"),
        (lambda: verify(most=1025), "most"), (lambda: verify(temp=-1.0), "temperature"), (lambda: verify(temp=float("inf")), "temperature"),
        (lambda: verify(temp=float("nan")), "temperature"), (lambda: verify(temp=1.0), "accept and pick"),
        (lambda: verify(temp=1.0, accept=fed), "go together"), (lambda: verify(temp=1.0, accept=one, pick=one), "one number"),
        (lambda: verify(temp=1.0, accept=fed, pick=fed), "one number"), (lambda: verify(draft=T(10, 3)), "draft's logits"),
        (lambda: verify(token_major=True), "one token"),
    ]


def test_refusals(cpu):
    for i, (call, msg) in enumerate(refusals(cpu)):
        with pytest.raises(nnengine.EngineError, match=msg):
            call()
            print("not refused:", i)
