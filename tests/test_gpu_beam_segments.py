"""nnhip_beam_select where its first pass puts segments of neighbouring tokens aside (csrc/k_beam.hip): distances at the
edge of the range that is sorted at once, more segments than are kept in LDS, segments that grow, against the 64-bit form
(paged_helpers.select)."""
import numpy as np
import pytest

import paged_helpers as ph
from test_gpu_paged import check_select, run_select

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("beam_major,seg", [(False, 64), (True, 256)])
@pytest.mark.parametrize("group", [0, 2])
def test_select_at_the_last_distance(beam_major, seg, group):
    """The last one taken lies just under 32 below the best total. Its beam has logits of 50000, where float32 distances
    are off by up to 1/512, and measures 32; another beam's candidate, a little worse, measures less than 32."""
    n_seg, take = 80, 3
    x = np.full((3, 2, n_seg * seg), -200.0, np.float32)
    scores = np.zeros((3, 2), np.float32)
    for g in range(3):      # the others: the best three far apart
        x[g, 0, [0, 5 * seg]], x[g, 1, 7] = [0, -3], -1
    x[group] = -60.0
    x[group, 1] = 49900.0
    x[group, 0, 3], x[group, 0, 9 * seg + 2] = 0, -(32 - 1 / 1024)
    x[group, 1, 5], x[group, 1, 11 * seg + 4] = 50000, 50000 - 27 + 1 / 256
    scores[group, 1] = -(5 + 1 / 512 + 2.0 ** -12)
    want = ph.select(x, scores, None, take, 0)
    assert want[1, group, 2] == 2 * group + 1 and -32 < want[0, group, 2] < -31.99
    check_select(run_select(x, scores, None, take, 0, beam_major), want)


def many_segments(beams, vocab, chunk, seed):
    """Logits of one group whose segments grow past what a thread or 16 lanes load at once (chunk tokens); the first
    beams, which have the best scores, end in every way: chunks of -inf behind a finite one, before it, around it, a NaN
    and a +inf in a later chunk, nothing but -inf, nothing finite but the last token."""
    rng = np.random.default_rng(seed)
    x = rng.normal(0, 3, (1, beams, vocab)).astype(np.float32)
    scores = rng.uniform(-12, -4, (1, beams)).astype(np.float32)
    if beams > 8:
        scores[0, :8] = rng.uniform(-1, 0, 8)
        x[0, 0, chunk:2 * chunk] = -np.inf
        x[0, 1, :chunk] = -np.inf
        x[0, 2, :2 * chunk] = x[0, 2, 3 * chunk:] = -np.inf
        x[0, 3, 2 * chunk - 1] = np.nan
        x[0, 4, chunk + 1] = np.inf
        x[0, 5] = -np.inf
        x[0, 6, :-1] = -np.inf
        x[0, 7, ::2] = -3.4028234663852886e38
    return x, scores


@pytest.mark.parametrize("beam_major,beams,vocab,take,seed", [
    (False, 32, 20011, 64, 2),     # 10016 segments: their bins do not fit in LDS
    (True, 40, 60001, 256, 2),     # 9400 segments of a row
    (False, 256, 16001, 256, 7),   # segments of two chunks, the last one cut
    (True, 140, 60001, 256, 1),    # segments of two chunks, rows
    (False, 1024, 5000, 256, 2),   # segments of four chunks
    (False, 1, 700001, 100, 2),    # one beam, 10938 segments
])
@pytest.mark.parametrize("ended", [False, True])
def test_select_many_segments(beam_major, beams, vocab, take, seed, ended):
    x, scores = many_segments(beams, vocab, 256 if beam_major else 64, seed)
    eos = vocab - 3
    done = None
    if ended:
        done = np.zeros((1, beams), np.float32)
        done[0, beams // 2:beams // 2 + 3] = 1
        scores[done != 0] += 8
    want = ph.select(x, scores, done, take + 1, eos)
    # Totals that are compared: off by what check_select allows and 6 2^-24 more for each part of a segment (a factor
    # of two exp's, products, a sum), and a rounding of totals of at most 16; the inputs keep those of different beams
    # further apart, and a beam's own are ordered exactly.
    tol = (70 + 6 * 4) * U + U * 16
    fin = want[0, 0][np.isfinite(want[0, 0])]
    assert np.abs(fin).max() <= 16
    near = np.nonzero(fin[:-1] - fin[1:] <= 2 * tol)[0]
    assert np.all(want[1, 0, near] == want[1, 0, near + 1])
    want = want[:, :, :take]
    got = run_select(x, scores, done, take, eos, beam_major)
    assert np.array_equal(got[1:], want[1:])
    ok = np.isfinite(want[0])
    assert np.all(np.abs(got[0][ok] - want[0][ok]) <= tol) and np.array_equal(got[0][~ok], want[0][~ok])
    if beams > 8:
        assert not set(got[1, 0][np.isfinite(got[0, 0])]) & {3, 4, 5} and {0, 1, 2, 7} <= set(got[1, 0])
