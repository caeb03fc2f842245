"""GPU: packed rows of more queries than max_q: the first max_q of each, at the positions that the whole row gives them."""

import pytest
import torch

from tests._window_cases import Case
from yapd_amd import kernels

pytestmark = pytest.mark.gpu

# (queries, keys, heads, window, sinks, max_q)
LONGER = [
    ([10], [10], 4, 100, 0, 8),
    ([10, 3, 9, 0, 40], [10, 3, 50, 7, 300], 8, 12, 2, 4),           # short tiles
    ([10] * 90, [10 + i for i in range(90)], 4, 30, 1, 6),
    ([64, 20], [200, 300], 4, 90, 5, 33),
    ([5, 2], [9000, 700], 4, 8000, 20, 2),                           # short tiles in parts, joined
    ([100], [150], 4, 33, 3, 70),                                    # tiles of 128: a single row
    ([300, 3, 190, 129], [900, 3, 190, 140], 4, 77, 3, 150),         # few rows: tiles dealt by weight
    ([90] * 70, [90 + 2 * i for i in range(70)], 4, 50, 4, 65),      # more rows than lanes
    ([400], [9000], 4, 8000, 16, 160),                               # tiles of 128 in parts, joined
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("q,kv,H,window,sinks,max_q", LONGER)
def test_rows_longer_than_max_q(dev, q, kv, H, window, sinks, max_q, causal):
    c = Case(q_lens=q, kv_lens=kv, H=H, window=window, sinks=sinks, causal=causal, packed=True, tail_q=2)
    out = c.run(dev, kernels, max_q=max_q).cpu().double()
    for r, n in enumerate(q):
        a, b = c.starts[r], c.starts[r] + min(n, max_q)
        assert bool(((out[a:b] - c.ref[a:b]).abs() <= c.tol[a:b]).all()), r
        assert bool((out[b:c.starts[r + 1]] == 77.0).all()), r
    assert bool((out[c.starts[-1]:] == 77.0).all())
