"""The bars of tests/score_bars.py and its rows against mistakes planted in the reference: an element lost or
counted twice at any edge moves the sums far past the bars."""
import numpy as np
import pytest

from score_bars import edge_positions, edge_row, sharp_bars
from score_ref import score_ref


@pytest.mark.parametrize("V", [50257, 16383, 60001, 151936])
@pytest.mark.parametrize("elem", [2, 4])
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_a_lost_or_doubled_element_is_seen(V, elem, offset):
    x, at = edge_row(V, elem, offset)
    _, h, _, log_sum, *_ = score_ref(x[None], None)
    bar, ebar = sharp_bars(x[None], 1.0, elem)
    for i in sorted({*at[:18], *at[-18:], *at[18:-18:7]}):
        lost = np.delete(x, i)
        for y in (lost, np.append(x, x[i])):
            _, h2, _, log_sum2, *_ = score_ref(y[None], None)
            assert abs(log_sum2 - log_sum)[0] > 20 * bar[0] and abs(h2 - h)[0] > 2 * ebar[0]
    # A tail of a few elements, as a kernel that stops at the last whole vector would lose it.
    _, h2, _, log_sum2, *_ = score_ref(x[None, :V - 3], None)
    assert log_sum[0] - log_sum2[0] > 100 * bar[0]


def test_edges_of_a_row():
    assert list(edge_positions(5, 4, 0)) == [0, 1, 2, 3, 4]
    at = edge_positions(50257, 2, 1)
    assert {0, 6, 7, 14, 50256, 7 + 2048, 7 + 2047, 7 + 2048 + 7} <= set(at.tolist())
    x, at = edge_row(50257, 2, 1)
    p = np.exp(x - x.max())
    assert p[at].sum() / p.sum() > 1 - 1e-8
