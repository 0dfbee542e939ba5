"""attn_chunk8 over rows that were not finite when they were stored, and queries that are not: NaN where a token sees them,
whatever weight they have."""
import numpy as np
import pytest


def rows_not_finite(e, which, at):
    """Six tokens of one sequence, the first with all of the weight; a key or value of token `at` is infinite. O (tokens, 4)
    over 8 bits."""
    rng = np.random.default_rng(at)
    k, v, q = (rng.normal(size=(4, 6)).astype(np.float32) for _ in range(3))
    k[0] = -300
    k[0, 0], q[0] = 300, 8
    (k if which == "k" else v)[2, at] = np.inf
    pos = np.arange(6, dtype=np.float32)[:, None]
    cache, table = e.kv8_cache(3, 4, 1, 4), e.tensor(np.array([[2, 0]], np.float32))
    e.kv8_append(cache, table, e.tensor(k), e.tensor(v), e.tensor(pos), 4, 1, 4, seq=e.tensor(np.zeros((6, 1), np.float32)))
    O = e.attn_chunk8(cache, table, e.tensor(q), e.tensor(np.array([[0.0], [6.0]], np.float32)), e.tensor(np.array([[6.0]], np.float32)),
                      6, 1.0, 4, 1, 4).numpy().T
    # The first token's value, as a byte holds it, is all that the others see.
    assert np.all(np.abs(O[:at] - v[:, 0]) <= np.abs(v[:, 0]).max() * (0.5 / 127 + 2.0 ** -20))
    assert np.isnan(O[at:]).all()


def queries_not_finite(e, bits):
    """Of three tokens the first sees itself alone, so that all of its scores are NaN."""
    rng = np.random.default_rng(bits)
    k, v, q = (rng.normal(size=(4, 3)).astype(np.float32) for _ in range(3))
    q[1, 0] = np.nan
    pos, seq = np.arange(3, dtype=np.float32)[:, None], np.zeros((3, 1), np.float32)
    table, start, lens = e.tensor(np.zeros((1, 1), np.float32)), e.tensor(np.array([[0.0], [3.0]], np.float32)), e.tensor(np.array([[3.0]], np.float32))
    if bits == 8:
        cache = e.kv8_cache(1, 4, 1, 4)
        e.kv8_append(cache, table, e.tensor(k), e.tensor(v), e.tensor(pos), 4, 1, 4, seq=e.tensor(seq))
        O = e.attn_chunk8(cache, table, e.tensor(q), start, lens, 3, 1.0, 4, 1, 4)
    else:
        K, V = (e.tensor(np.zeros((4, 4), np.float32)) for _ in range(2))
        e.kv_append(K, V, table, e.tensor(k), e.tensor(v), e.tensor(pos), 4, 1, seq=e.tensor(seq))
        O = e.attn_chunk(K, V, table, e.tensor(q), start, lens, 3, 1.0, 4, 1)
    O = O.numpy().T
    assert np.isnan(O[0]).all() and np.isfinite(O[1:]).all()


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("at", [1, 3, 5])
def test_rows_not_finite(cpu, which, at):
    rows_not_finite(cpu, which, at)


@pytest.mark.parametrize("bits", [32, 8])
def test_queries_not_finite(cpu, bits):
    queries_not_finite(cpu, bits)
