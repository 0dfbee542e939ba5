"""What the paged-cache and beam-search entry points refuse, and the calls that have nothing to do. Every check is
made on the host before any launch, so these run without a GPU; the pointers are never followed."""
import pytest

from paged_helpers import Pages, library

P = 4096   # a pointer's stand-in, aligned


def pages(**kw):
    d = dict(K=P, V=1 << 24, table=P, batch=4, width=8, pages=16, page=16, heads=4, dim=64, row=256)
    d.update(kw)
    return Pages(**d)


BAD_PAGES = [dict(K=None), dict(V=None), dict(table=None), dict(batch=0), dict(width=0), dict(pages=0), dict(page=0),
             dict(heads=0), dict(dim=0), dict(row=255), dict(pages=(1 << 24) + 1), dict(batch=(1 << 24) + 1),
             dict(width=1 << 21, page=16), dict(pages=1 << 20, page=1 << 11), dict(width=1 << 63, page=2), dict(dim=257, row=4 * 257)]


def append(c, **kw):
    a = dict(k=P, v=P, q=P, out=P, st=(1, 4), q_heads=4, tokens=4, seq=P, pos=P, cos=P, sin=P, rows=8, rope=64)
    a.update(kw)
    s = a["st"]
    return library().nnhip_kv_append(c, a["k"], *s, a["v"], *s, a["q"], *s, a["out"], *s, a["q_heads"], a["tokens"],
                                     a["seq"], a["pos"], a["cos"], a["sin"], a["rows"], a["rope"], None)


@pytest.mark.parametrize("bad", BAD_PAGES)
def test_append_pages(bad):
    assert append(pages(**bad)) == -1


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(pos=None), dict(q=None), dict(out=None), dict(q_heads=0),
                                 dict(st=(-1, 4)), dict(st=(1, -4)), dict(cos=None), dict(sin=None), dict(rope=63),
                                 dict(rope=66), dict(rope=0), dict(rows=0), dict(cos=None, sin=None),
                                 dict(tokens=(1 << 24) + 1), dict(q_heads=70000), dict(rows=(1 << 24) + 1)])
def test_append_arguments(bad):
    assert append(pages(), **bad) == -1


def test_append_keys_over_values():
    assert append(pages(V=P)) == -1


def test_append_of_nothing():
    assert append(pages(), tokens=0, k=None) == 0
    assert append(None) == -1


def attend(c, **kw):
    a = dict(q=P, st=(256, 1), q_heads=4, len=P, shared=P, group=2, O=P, ws=P, nbytes=1 << 40)
    a.update(kw)
    s = a["st"]
    return library().nnhip_attn_paged(c, a["q"], *s, a["q_heads"], a["len"], a["shared"], a["group"], None, 1.0, a["O"], *s,
                                      None, None, a["ws"], a["nbytes"], None)


@pytest.mark.parametrize("bad", BAD_PAGES + [dict(dim=129, row=4 * 129)])
def test_attend_pages(bad):
    assert attend(pages(**bad)) == -1
    assert library().nnhip_attn_paged_workspace_bytes(pages(**bad), 4, 2) == 0


@pytest.mark.parametrize("bad", [dict(q=None), dict(len=None), dict(O=None), dict(q_heads=0), dict(q_heads=6), dict(group=0),
                                 dict(group=3), dict(group=8), dict(st=(-1, 1)), dict(st=(1, -1)), dict(ws=None),
                                 dict(ws=P + 8), dict(nbytes=0)])
def test_attend_arguments(bad):
    need = library().nnhip_attn_paged_workspace_bytes(pages(), 4, 2)
    assert need > 0
    assert attend(pages(), **bad) == -1
    assert attend(pages(), nbytes=need - 1) == -1
    assert attend(None) == -1


def select(**kw):
    a = dict(logits=P, ld=4, bm=0, scores=P, done=P, groups=2, beams=2, vocab=100, take=4, eos=5, o=(P, P, P), ws=P,
             nbytes=1 << 40)
    a.update(kw)
    return library().nnhip_beam_select(a["logits"], a["ld"], a["bm"], a["scores"], a["done"], a["groups"], a["beams"],
                                       a["vocab"], a["take"], a["eos"], *a["o"], a["ws"], a["nbytes"], None)


@pytest.mark.parametrize("bad", [dict(logits=None), dict(scores=None), dict(o=(None, P, P)), dict(o=(P, None, P)),
                                 dict(o=(P, P, None)), dict(beams=0), dict(vocab=0), dict(take=0), dict(take=257),
                                 dict(vocab=1, take=3, eos=0), dict(ld=3), dict(bm=1, ld=99), dict(eos=100), dict(ws=None),
                                 dict(nbytes=8), dict(ws=P + 4), dict(beams=1025, ld=4000), dict(vocab=(1 << 24) + 1),
                                 dict(groups=1 << 23, beams=4, ld=1 << 30), dict(groups=1, beams=1000, ld=1000, vocab=1 << 22)])
def test_select_arguments(bad):
    assert select(**bad) == -1


def test_select_of_nothing():
    assert select(groups=0, logits=None) == 0


def reorder(layers, n=None, **kw):
    a = dict(parent=2 * P, len=3 * P, fresh=4 * P, out_batch=4, out=1 << 20, out_len=1 << 21)
    a.update(kw)
    arr = (Pages * len(layers))(*layers)
    return library().nnhip_kv_reorder(arr, len(layers) if n is None else n, a["parent"], a["len"], a["fresh"],
                                      a["out_batch"], a["out"], a["out_len"], None)


@pytest.mark.parametrize("bad", [b for b in BAD_PAGES if "dim" not in b or b["dim"] == 0])
def test_reorder_pages(bad):
    assert reorder([pages(**bad)]) == -1
    assert reorder([pages(), pages(**bad)]) == -1


@pytest.mark.parametrize("bad", [dict(parent=None), dict(len=None), dict(out=None), dict(out_len=None),
                                 dict(out_batch=(1 << 24) + 1), dict(out=P), dict(out=P + 4 * 31), dict(out=P - 4 * 31),
                                 dict(out_len=3 * P), dict(out_len=3 * P + 12), dict(out_len=2 * P - 12), dict(out_len=4 * P),
                                 dict(out=2 * P), dict(out=4 * P - 4 * 31)])
def test_reorder_arguments(bad):
    assert reorder([pages()], **bad) == -1


def test_reorder_layers():
    assert reorder([pages()], n=0) == -1
    assert reorder([pages()], out_batch=0, parent=None) == 0
    for other in (dict(table=2 * P), dict(batch=5), dict(width=9), dict(pages=17), dict(page=8), dict(heads=2),
                  dict(dim=32), dict(row=512)):
        assert reorder([pages(), pages(**other)]) == -1


@pytest.mark.parametrize("bad", [dict(out=3 * P), dict(out=3 * P - 4 * 31), dict(out=3 * P + 12), dict(out_len=P), dict(out_len=P - 12),
                                 dict(out_len=P + 4 * 31), dict(out_len=1 << 20), dict(out_len=(1 << 20) + 4 * 31),
                                 dict(out_len=(1 << 20) - 12), dict(out=P + (1 << 18) - 4), dict(out=(1 << 24) + (1 << 17)),
                                 dict(out_len=P + (1 << 18) - 4), dict(out_len=(1 << 24) - 12)])
def test_reorder_outputs_over_the_rest(bad):
    """The table's output on the lengths, the lengths' on the table, one output on the other, either on the caches."""
    assert reorder([pages()], **bad) == -1


@pytest.mark.parametrize("heads,dim", [(1 << 8, 1 << 24), (255, 1 << 24), (1 << 9, 1 << 23), (1 << 7, 1 << 24)])
def test_reorder_rows_past_31_bits(heads, dim):
    """Rows of 2^31 values and more: the kernel counts a row's values in 32 bits, up to 256 past the last."""
    assert reorder([pages(K=1 << 48, V=1 << 56, heads=heads, dim=dim, row=heads * dim, pages=1, page=1)]) == -1


@pytest.mark.parametrize("batch,q_heads", [(1 << 20, 16), (1 << 21, 8), (1 << 24, 1), ((1 << 20) - 16, 16)])
def test_attend_more_workgroups_than_a_grid_has(batch, q_heads):
    """A workgroup of 256 a sequence and key head, and a grid of fewer than 2^32 threads. One short of that is not refused."""
    refused = batch * q_heads >= 1 << 24
    rc = attend(pages(batch=batch, width=1, heads=q_heads, row=64 * q_heads), q_heads=q_heads, shared=None, group=1)
    assert (rc == -1) == refused


def test_reorder_more_workgroups_than_a_grid_has():
    big = dict(K=1 << 50, V=1 << 54, table=1 << 58, page=1, pages=16)
    assert reorder([pages(batch=1 << 10, width=1 << 22, **big)], out_batch=1 << 10, out=1 << 44, out_len=1 << 43) == -1
    assert reorder([pages(batch=1 << 10, width=1 << 21, **big)], out_batch=1 << 10, out=1 << 44, out_len=1 << 43) != -1
    assert reorder([pages(batch=4, width=8, **dict(big, page=2))] * 32, out_batch=1 << 18, out=1 << 44, out_len=1 << 43) == -1


def test_reorder_outputs_behind_the_caches():
    """Values interleaved with keys, V behind K's heads in rows of twice their width: an output right behind the last row
    is not on it, one on its last value is."""
    kv = dict(K=1 << 30, V=(1 << 30) + 4 * 256, row=512)
    end = (1 << 30) + 4 * 512 * 16 * 16
    for at, refused in ((end, False), (end - 4, True), ((1 << 30) - 4 * 32, False), ((1 << 30) - 4 * 31, True)):
        assert (reorder([pages(**kv)], out=at) == -1) == refused
        assert (reorder([pages(**kv), pages(**kv)], out=at) == -1) == refused
