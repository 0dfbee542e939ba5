"""What the 8-bit caches, chunk attention and draft verification refuse, and the calls that have nothing to do. Every check
is made on the host before any launch, so these run without a GPU; the pointers are never followed."""
import pytest

from chunk_helpers import Pages, Pages8, library

P = 4096   # a pointer's stand-in, aligned
SIZES = dict(batch=4, width=8, pages=16, page=16, heads=4, dim=64, row=256)


def pages(**kw):
    return Pages(**dict(dict(K=P, V=1 << 24, table=P, **SIZES), **kw))


def pages8(**kw):
    return Pages8(**dict(dict(K=P, V=1 << 24, K_scale=1 << 25, V_scale=1 << 26, table=P, **SIZES), **kw))


BAD_PAGES = [dict(K=None), dict(V=None), dict(table=None), dict(batch=0), dict(width=0), dict(pages=0), dict(page=0),
             dict(heads=0), dict(dim=0), dict(row=255), dict(pages=(1 << 24) + 1), dict(batch=(1 << 24) + 1),
             dict(width=1 << 21, page=16), dict(pages=1 << 20, page=1 << 11), dict(width=1 << 63, page=2), dict(dim=257, row=4 * 257)]
BAD_SCALES = [dict(K_scale=None), dict(V_scale=None)]


def store(c, **kw):
    a = dict(k=P, v=P, q=P, out=P, st=(1, 4), q_heads=4, tokens=4, seq=P, pos=P, cos=P, sin=P, rows=8, rope=64)
    a.update(kw)
    s = a["st"]
    return library().nnhip_kv8_append(c, a["k"], *s, a["v"], *s, a["q"], *s, a["out"], *s, a["q_heads"], a["tokens"],
                                      a["seq"], a["pos"], a["cos"], a["sin"], a["rows"], a["rope"], None)


@pytest.mark.parametrize("bad", BAD_PAGES + BAD_SCALES + [dict(V=P), dict(V_scale=1 << 25), dict(K_scale=P), dict(V_scale=1 << 24),
                                                          dict(V_scale=P), dict(K_scale=1 << 24)])
def test_store_pages(bad):
    assert store(pages8(**bad)) == -1


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(pos=None), dict(q=None), dict(out=None), dict(q_heads=0),
                                 dict(st=(-1, 4)), dict(st=(1, -4)), dict(cos=None), dict(sin=None), dict(rope=63),
                                 dict(rope=66), dict(rope=0), dict(rows=0), dict(cos=None, sin=None),
                                 dict(tokens=(1 << 24) + 1), dict(q_heads=70000), dict(rows=(1 << 24) + 1)])
def test_store_arguments(bad):
    assert store(pages8(), **bad) == -1


def test_store_of_nothing():
    assert store(pages8(), tokens=0, k=None) == 0
    assert store(None) == -1


def read(c, **kw):
    a = dict(k=P, v=P, st=(1, 4), tokens=4, seq=P, pos=P)
    a.update(kw)
    return library().nnhip_kv8_read(c, a["k"], *a["st"], a["v"], *a["st"], a["tokens"], a["seq"], a["pos"], None)


@pytest.mark.parametrize("bad", BAD_PAGES + BAD_SCALES)
def test_read_pages(bad):
    assert read(pages8(**bad)) == -1


@pytest.mark.parametrize("bad", [dict(pos=None), dict(st=(-1, 4)), dict(st=(1, -4)), dict(tokens=(1 << 24) + 1)])
def test_read_arguments(bad):
    assert read(pages8(), **bad) == -1
    assert read(pages8(heads=1 << 15, row=64 << 15)) == -1
    assert read(pages8(), tokens=0, pos=None) == 0
    assert read(pages8(), k=None, v=None, pos=None) == 0
    assert read(None) == -1


def chunk(c, **kw):
    a = dict(q=P, st=(256, 1), q_heads=4, tokens=8, start=P, most=3, len=P, O=P, ws=P, nbytes=1 << 50)
    a.update(kw)
    s = a["st"]
    f = library().nnhip_attn_chunk if isinstance(c, Pages) else library().nnhip_attn_chunk8
    return f(c, a["q"], *s, a["q_heads"], a["tokens"], a["start"], a["most"], a["len"], None, 1.0, a["O"], *s, None, None, a["ws"],
             a["nbytes"], None)


@pytest.mark.parametrize("make", [pages, pages8])
@pytest.mark.parametrize("bad", BAD_PAGES + [dict(dim=129, row=4 * 129)])
def test_chunk_pages(make, bad):
    assert chunk(make(**bad)) == -1
    f = library().nnhip_attn_chunk_workspace_bytes if make is pages else library().nnhip_attn_chunk8_workspace_bytes
    assert f(make(**bad), 4, 8, 3) == 0


@pytest.mark.parametrize("make", [pages, pages8])
@pytest.mark.parametrize("bad", [dict(q=None), dict(start=None), dict(len=None), dict(O=None), dict(q_heads=0), dict(q_heads=6),
                                 dict(tokens=0), dict(most=0), dict(most=9), dict(st=(-1, 1)), dict(st=(1, -1)), dict(ws=None),
                                 dict(ws=P + 8), dict(nbytes=0), dict(tokens=1 << 24, q_heads=128), dict(tokens=(1 << 24) + 1)])
def test_chunk_arguments(make, bad):
    f = library().nnhip_attn_chunk_workspace_bytes if make is pages else library().nnhip_attn_chunk8_workspace_bytes
    need = f(make(), 4, 8, 3)
    assert need > 0
    assert chunk(make(), **bad) == -1
    assert chunk(make(), nbytes=need - 1) == -1


@pytest.mark.parametrize("bad", BAD_SCALES)
def test_chunk_scales(bad):
    assert chunk(pages8(**bad)) == -1


@pytest.mark.parametrize("make", [pages, pages8])
def test_chunk_more_workgroups_than_a_grid_has(make):
    big = dict(batch=1 << 20, width=1, heads=16, row=64 * 16)
    assert chunk(make(**big), q_heads=16, tokens=1 << 20, most=1) == -1
    assert chunk(make(**dict(big, batch=1 << 24)), q_heads=16, tokens=1 << 20, most=1) == -1


def verify(**kw):
    a = dict(target=P, t_ld=8, draft=P, d_ld=8, tm=0, vocab=100, tokens=8, fed=P, start=P, batch=2, most=4, T=1.0, accept=P, pick=P,
             o=(P, P), ws=P, nbytes=1 << 50)
    a.update(kw)
    return library().nnhip_draft_verify(a["target"], a["t_ld"], a["draft"], a["d_ld"], a["tm"], a["vocab"], a["tokens"], a["fed"],
                                        a["start"], a["batch"], a["most"], a["T"], a["accept"], a["pick"], *a["o"], a["ws"],
                                        a["nbytes"], None)


@pytest.mark.parametrize("bad", [dict(target=None), dict(fed=None), dict(start=None), dict(accept=None), dict(pick=None),
                                 dict(o=(None, P)), dict(o=(P, None)), dict(t_ld=7), dict(d_ld=7), dict(tm=1, t_ld=99, d_ld=100),
                                 dict(tm=1, t_ld=100, d_ld=99), dict(vocab=0), dict(vocab=(1 << 24) + 1), dict(tokens=0),
                                 dict(tokens=(1 << 24) + 1), dict(batch=(1 << 24) + 1), dict(most=0), dict(most=1025), dict(T=-0.5),
                                 dict(T=float("nan")), dict(T=float("inf")), dict(ws=None), dict(ws=P + 8), dict(nbytes=0),
                                 dict(t_ld=(1 << 32) + 1), dict(batch=1 << 23, vocab=32000)])
def test_verify_arguments(bad):
    need = library().nnhip_draft_verify_workspace_bytes(8, 2, 4, 100)
    assert need > 0
    assert verify(**bad) == -1
    assert verify(nbytes=need - 1) == -1
    assert verify(batch=0, target=None) == 0


def test_verify_workspace_of_nothing():
    f = library().nnhip_draft_verify_workspace_bytes
    assert f(0, 2, 4, 100) == f(8, 0, 4, 100) == f(8, 2, 0, 100) == f(8, 2, 4, 0) == f(8, 2, 1025, 100) == 0
