"""nnhip_attn_chunk and nnhip_attn_chunk8 where most tokens belong to no sequence."""
import numpy as np
import pytest

import chunk_helpers as ch
from test_gpu_chunk import cache_for, check_chunk, run_chunk

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("new,past,heads,per,dim", [([3, 1], [500, 90], 1, 2, 64), ([1], [3000], 2, 4, 128), ([2, 0, 8], [40, 7, 2000], 2, 4, 40),
                                                    ([1, 1, 40, 1], [900, 3, 700, 50], 1, 2, 64), ([8], [200], 2, 4, 30)])
def test_tokens_of_no_sequence(new, past, heads, per, dim, bits):
    rng = np.random.default_rng(sum(past))
    page, tokens, first = 16, 2000, 700
    lens, start = [n + p for n, p in zip(new, past)], first + np.concatenate([[0], np.cumsum(new)])
    x, table, pages = cache_for(rng, lens, page, heads, dim, bits)
    q = rng.normal(size=(tokens, heads * per, dim)).astype(np.float32)
    c = dict(pages=pages, page=page, heads=heads, dim=dim)
    got = run_chunk(x, c, table, q, start, max(new), lens, None, 0.125)
    check_chunk(got, ch.attend(q, x["K64"], x["V64"], table, page, pages, heads, start, max(new), lens, 0.125))
