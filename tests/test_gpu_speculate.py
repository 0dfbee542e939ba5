"""Chunks of new tokens, 8-bit caches, drafted tokens and speculative decoding on the HIP engine (tests/test_speculate.py's
checks, and the CPU oracle's results)."""
import numpy as np
import pytest

import draft_reference
import nnengine
import test_speculate as cpu_tests

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed", [0, 1, 2])
def test_calls(hip, seed):
    cpu_tests.check_ops(*cpu_tests.run_ops(hip, seed))


def test_refusals(hip):
    for call, msg in cpu_tests.refusals(hip):
        with pytest.raises(nnengine.EngineError, match=msg):
            call()


def test_verified_tokens_follow_the_target(hip):
    cpu_tests.verified_distribution(hip)


@pytest.mark.parametrize("variant", cpu_tests.VARIANTS, ids=lambda v: v["pos_enc"])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("draft_len", [1, 4, 11])
def test_greedy(hip, variant, bits, draft_len):
    print(f"[speculate] {variant['pos_enc']} bits {bits} draft_len {draft_len}", flush=True)
    cpu_tests.greedy_run(hip, variant, bits, draft_len)


@pytest.mark.parametrize("bits", [32, 8])
def test_distribution(hip, bits):
    cpu_tests.distribution(hip, bits)


def test_session_refusals(hip):
    cpu_tests.session_refusals(hip)


def test_backward_needs_its_own_forward(hip):
    cpu_tests.backward_needs_its_own_forward(hip)


@pytest.mark.parametrize("bits", [32, 8])
def test_larger_model(hip, bits):
    """A 768-wide model with 12 heads and a 256-wide draft, prompts of several chunks: the tokens are the largest logits of a
    float64 pass, the same ones every time, whatever ran in between. Logits of 768 products of 0.05-wide gains and weights are
    0.07 wide: float32 changes them by 1e-6 of that, and a byte that it rounds the other way, a value by 1/127 of its head's
    largest (some 3.5 deviations) among 768, by 1e-3 of it: 2e-3 is a few dozen such bytes."""
    cfg = dict(vocab_size=1024, d_model=768, seq_len=1200, num_heads=12, d_ff=512, num_layers=2, pos_enc="rope")
    g, params = cpu_tests.session(hip, cfg, 6, 0.05)
    d, _ = cpu_tests.session(hip, dict(cfg, d_model=256, num_heads=4, d_ff=128, num_layers=1), 7, 0.05)
    rng = np.random.default_rng(bits)
    prompts = [rng.integers(0, 1024, n).tolist() for n in (40, 1, 700)]
    first = g.speculate(d, prompts, 9, 3, cache_bits=bits)
    clear = sum(draft_reference.check_greedy(f, params, p, 9, -1, cfg, bits, 2e-3) for f, p in zip(first[0], prompts))
    assert clear >= 20
    toks = rng.integers(0, 1024, (65, 1))
    step0 = [g.forward_step(int(t), i, i) for i, t in enumerate(toks[:5, 0])]
    assert g.speculate(d, prompts, 9, 3, cache_bits=bits) == first
    g.reset_cache()
    step1 = [g.forward_step(int(t), i, i) for i, t in enumerate(toks[:5, 0])]
    assert all(np.array_equal(a, b) for a, b in zip(step0, step1))
    drawn = g.speculate(d, prompts, 9, 3, temperature=1.0, seed=3, cache_bits=bits)
    assert g.speculate(d, prompts, 9, 3, temperature=1.0, seed=3, cache_bits=bits) == drawn


def test_slices_as_inputs(hip, cpu):
    """Tensors that are slices of others, and caches that were just zeroed or sliced before they are written."""
    def run(e):
        rng = np.random.default_rng(5)
        heads, d, page, pages, n = 2, 8, 4, 6, 10
        both = e.tensor(rng.normal(size=(80, n)).astype(np.float32))
        k, v, q = (e.slice_rows(both, i, heads * d) for i in (1, 17, 40))
        table = e.slice_rows(e.tensor(rng.permutation(24).reshape(4, 6).astype(np.float32) % pages), 1, 2)
        c8 = e.kv8_cache(pages, page, heads, d)
        before = e.slice_rows(c8[0], 0, 5)
        seq, pos = e.tensor((np.arange(n) % 2)[:, None]), e.tensor((np.arange(n) // 2)[:, None])
        e.kv8_append(c8, table, k, v, pos, page, heads, d, seq=seq)
        after = e.slice_rows(c8[0], 0, 24)
        order = e.tensor(np.argsort(np.arange(n) % 2, kind="stable")[:, None])
        qs = e.transpose(e.gather_rows(e.transpose(q), order))
        O = e.attn_chunk8(c8, table, qs, e.tensor([[0], [5], [10]]), e.tensor([[5], [5]]), 5, 0.5, page, heads, d)
        rk, rv = e.kv8_read(c8, table, pos, page, heads, d, seq=seq)
        return [t.numpy() for t in (before, after, O, rk, rv, both, *c8)]
    got, want = run(hip), run(cpu)
    assert not got[0].any()
    for i, (a, b) in enumerate(zip(got, want)):
        if i in (0, 1, 6, 7):
            assert np.array_equal(a.view(np.int8), b.view(np.int8))
        else:
            assert np.abs(a - b).max() <= 1e-5


def test_calls_between_graphs_and_streams(hip):
    """The four kernels' calls as one step of serving, captured once and replayed with other contents, eager work and a
    second step with its own workspaces on another stream in between: every replay equals the eager step."""
    import torch

    import chunk_helpers as ch
    from test_gpu_paged import dev, ptr
    lib = ch.library()
    B, n, qh, heads, dim, page, width, vocab = 3, 5, 8, 2, 64, 16, 30, 1000
    N, pages = B * n, B * width
    rng = np.random.default_rng(0)

    def state(seed):
        r = np.random.default_rng(seed)
        st = {k: torch.zeros(s).cuda() for k, s in dict(q=(N, qh * dim), qr=(N, qh * dim), k=(N, heads * dim), v=(N, heads * dim), o=(N, qh * dim),
                                                         kb=(N, heads * dim), vb=(N, heads * dim), target=(N, vocab), draft=(N, vocab),
                                                         fed=(N,), accept=(N,), pick=(B,), stand=(B,), token=(B,), lens=(B,), pos=(N,)).items()}
        st["K"], st["V"] = (torch.zeros(pages * page, heads * dim, dtype=torch.int8).cuda() for _ in range(2))
        st["Ks"], st["Vs"] = (torch.zeros(pages * page, heads).cuda() for _ in range(2))
        st["table"] = dev(r.permutation(pages).reshape(B, width).astype(np.float32))
        return st

    cos, sin = dev(rng.normal(size=(width * page, dim // 2))), dev(rng.normal(size=(width * page, dim // 2)))
    seq, start = dev(np.repeat(np.arange(B), n)), dev(np.arange(B + 1) * n)

    def bound(st):
        c = ch.Pages8(ptr(st["K"]), ptr(st["V"]), ptr(st["Ks"]), ptr(st["Vs"]), ptr(st["table"]), B, width, pages, page, heads, dim, heads * dim)
        n1, n2 = lib.nnhip_attn_chunk8_workspace_bytes(c, qh, N, n), lib.nnhip_draft_verify_workspace_bytes(N, B, n, vocab)
        w1, w2 = torch.full((n1 // 4 + 4,), float("nan")).cuda(), torch.full((n2 // 4 + 4,), float("nan")).cuda()

        def step():
            s = torch.cuda.current_stream().cuda_stream
            kd, qd = heads * dim, qh * dim
            assert lib.nnhip_kv8_append(c, ptr(st["k"]), kd, 1, ptr(st["v"]), kd, 1, ptr(st["q"]), qd, 1, ptr(st["qr"]), qd, 1, qh, N,
                                        ptr(seq), ptr(st["pos"]), ptr(cos), ptr(sin), width * page, dim, s) == 0
            assert lib.nnhip_attn_chunk8(c, ptr(st["qr"]), qd, 1, qh, N, ptr(start), n, ptr(st["lens"]), None, 0.125, ptr(st["o"]), qd, 1,
                                         None, None, ptr(w1), n1, s) == 0
            assert lib.nnhip_kv8_read(c, ptr(st["kb"]), kd, 1, ptr(st["vb"]), kd, 1, N, ptr(seq), ptr(st["pos"]), s) == 0
            assert lib.nnhip_draft_verify(ptr(st["target"]), vocab, ptr(st["draft"]), vocab, 1, vocab, N, ptr(st["fed"]), ptr(start), B, n, 0.9,
                                          ptr(st["accept"]), ptr(st["pick"]), ptr(st["stand"]), ptr(st["token"]), ptr(w2), n2, s) == 0
        return step

    def load(st, i):
        r = np.random.default_rng(100 + i)
        for k in ("q", "k", "v", "target"):
            st[k].copy_(dev(r.normal(size=tuple(st[k].shape))))
        st["draft"].copy_(st["target"] + 0.3 * dev(r.normal(size=(N, vocab))))
        st["fed"].copy_(dev(r.integers(0, vocab, N)))
        st["fed"][1::n] = st["target"][::n].argmax(1).float()
        st["accept"].copy_(dev(r.random(N)))
        st["pick"].copy_(dev(r.random(B)))
        past = dev(100 * i + 10 * np.arange(B))
        st["lens"].copy_(past + n)
        st["pos"].copy_((past[:, None] + torch.arange(n).cuda()[None, :]).reshape(-1))

    outs = ("K", "V", "Ks", "Vs", "qr", "o", "kb", "vb", "stand", "token")
    st, other = state(1), state(2)
    step, step2 = bound(st), bound(other)
    side, side2 = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        load(st, 0)
        step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
    torch.cuda.synchronize()
    for i in range(4):
        got = []
        for replay in (True, False):
            for k in ("K", "V", "Ks", "Vs"):
                st[k].zero_()
            load(st, i)
            load(other, i + 7 if replay else i)
            torch.cuda.synchronize()
            with torch.cuda.stream(side2):
                step2()
            if replay:
                graph.replay()
            else:
                step()
            torch.cuda.synchronize()
            got.append({k: st[k].clone() for k in outs})
        for k in outs:
            assert torch.equal(got[0][k], got[1][k]), (i, k)
        assert got[0]["o"].abs().sum() > 0


@pytest.mark.parametrize("bits", [32, 8])
def test_prompts_in_a_graph(hip, bits):
    """A prompt's chunk beside single tokens, every kernel of the attention, captured and replayed with other contents and
    lengths: the same bits as the eager calls."""
    import torch

    import chunk_helpers as ch
    from test_gpu_paged import dev, ptr
    lib = ch.library()
    new, qh, heads, dim, page, width = [70, 1, 1, 40], 4, 2, 64, 16, 40
    B, N, pages = len(new), sum(new), len(new) * width
    rng = np.random.default_rng(bits)
    table, start = dev(rng.permutation(pages).reshape(B, width)), dev(np.concatenate([[0], np.cumsum(new)]))
    q, o, lens = torch.zeros(N, qh * dim).cuda(), torch.zeros(N, qh * dim).cuda(), torch.zeros(B).cuda()
    if bits == 32:
        K, V = (torch.zeros(pages * page, heads * dim).cuda() for _ in range(2))
        c = ch.Pages(ptr(K), ptr(V), ptr(table), B, width, pages, page, heads, dim, heads * dim)
        need, call = lib.nnhip_attn_chunk_workspace_bytes(c, qh, N, 70), lib.nnhip_attn_chunk
    else:
        K, V = (torch.zeros(pages * page, heads * dim, dtype=torch.int8).cuda() for _ in range(2))
        Ks, Vs = (torch.zeros(pages * page, heads).cuda() for _ in range(2))
        c = ch.Pages8(ptr(K), ptr(V), ptr(Ks), ptr(Vs), ptr(table), B, width, pages, page, heads, dim, heads * dim)
        need, call = lib.nnhip_attn_chunk8_workspace_bytes(c, qh, N, 70), lib.nnhip_attn_chunk8
    ws = torch.full((need // 4 + 4,), float("nan")).cuda()

    def step():
        assert call(c, ptr(q), qh * dim, 1, qh, N, ptr(start), 70, ptr(lens), None, 0.125, ptr(o), qh * dim, 1, None, None, ptr(ws), need,
                    torch.cuda.current_stream().cuda_stream) == 0

    def load(i):
        r = np.random.default_rng(50 + i)
        q.copy_(dev(r.normal(size=(N, qh * dim))))
        lens.copy_(dev(np.array(new) + [100 * i, 30, 500 - 100 * i, 0]))
        for t in (K, V):
            t.copy_(dev(r.normal(size=tuple(t.shape))) if bits == 32 else torch.as_tensor(r.integers(-127, 128, tuple(t.shape)).astype(np.int8)).cuda())
        if bits == 8:
            for t in (Ks, Vs):
                t.copy_(dev(r.uniform(0.005, 0.02, tuple(t.shape))))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        load(0)
        step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
    torch.cuda.synchronize()
    for i in range(4):
        got = []
        for replay in (True, False):
            load(i)
            o.fill_(3.0)
            torch.cuda.synchronize()
            graph.replay() if replay else step()
            torch.cuda.synchronize()
            got.append(o.clone())
        assert torch.equal(*got) and got[0].abs().sum() > 0
