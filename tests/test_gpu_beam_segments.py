"""nnhip_beam_select where its first pass puts segments of neighbouring tokens aside (csrc/k_beam.hip): distances at the
edge of the range that is sorted at once, against the 64-bit form (paged_helpers.select)."""
import numpy as np
import pytest

import paged_helpers as ph
from test_gpu_paged import check_select, run_select

pytestmark = pytest.mark.gpu


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
