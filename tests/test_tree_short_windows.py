"""Packed trees behind windows shorter than the most nodes a row may have: the bound of the rows' nodes (64 unless given)
says nothing about the rows, so the same rows are taken whatever the batch's size."""

import pytest
import torch

from tests._tree_cases import Case
from yapd_amd import kernels

P = 4096  # never read: refused calls launch nothing


def tree(**over):
    a = dict(q=P, tok=1024, pool=P, bits=8, pages=100, table=P, stride=8, cols=8, kv_len=P, q_start=P, mask=P, rows=2,
             max_q=3, n_q=6, heads=16, window=2, sinks=0, max_kv=100, scale=0.0, ws=None, floats=0, out=1 << 40, stream=None)
    a.update(over)
    return list(a.values())


@pytest.mark.parametrize("over,msg", [(dict(), b"scale"), (dict(window=0), b"window >= 1"), (dict(sinks=-1), b"window"),
                                      (dict(q_start=None), b"window >= max_q")])
def test_refusals(over, msg):
    """A packed call's window is only refused below 1 (here the scale is refused next); with max_q nodes in every row below max_q."""
    lib = kernels.load_library()
    assert lib.yapd_attn_tree(*tree(**over)) == 1
    assert msg in lib.yapd_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("n,kv,H,window,sinks,kind", [
    ([1] * 70, [1 + 7 * i for i in range(70)], 8, 16, 4, "tree"),               # a batch of single tokens
    ([1] * 3, [900, 70, 1], 4, 1, 0, "tree"),                                   # themselves alone
    ([20, 64, 1, 33], [20, 200, 90, 300], 4, 7, 3, "chain"),                    # deeper than the window
    ([20, 64, 1, 33], [20, 200, 90, 300], 4, 25, 40, "tree"),
    ([3, 64, 0, 7], [3000, 64, 0, 2500], 4, 5, 2900, "padded"),                 # sinks long enough for parts
])
def test_packed_rows(dev, n, kv, H, window, sinks, kind, bits):
    c = Case(n_nodes=n, kv_lens=kv, H=H, bits=bits, window=window, sinks=sinks, kind=kind, seed=len(n), packed=True, tail_q=2)
    c.check(c.run(dev, kernels))


@pytest.mark.gpu
def test_the_bound_of_nodes_does_not_change_a_result_beyond_rounding(dev):
    c = Case(n_nodes=[1] * 66, kv_lens=[40 + 3 * i for i in range(66)], H=4, bits=8, window=20, sinks=2, packed=True)
    c.check(c.run(dev, kernels))
    c.check(c.run(dev, kernels, max_q=1))
    t = c.device(dev)
    with pytest.raises(ValueError, match="window"):
        kernels.attn_tree(t["q"], t["pool"], t["table"], t["kv_len"], t["mask"], torch.empty_like(t["q"]), 0.125, window=0,
                          q_start=t["q_start"])
