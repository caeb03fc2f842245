"""GPU: page copies against torch's index operations, and the shared paged cache against a plain model."""

import numpy as np
import pytest
import torch

from tests._shared_kv_model import Model, play
from yapd_amd import kernels
from yapd_amd.paged import PagedKV, SharedPagedKV

pytestmark = pytest.mark.gpu


def pools_of(dev, layers, pages, heads, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return [torch.randint(-2**15, 2**15, (pages, 2, heads, 1024), generator=g, device=dev, dtype=torch.int16)
            .view(torch.bfloat16) for _ in range(layers)]  # any bits, NaN among them


def same(a, b):
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.parametrize("layers,heads,pages,n", [(1, 4, 2, 1), (30, 16, 40, 1), (3, 16, 40, 20), (2, 20, 11, 5),
                                                  (1, 4, 800, 399), (65, 4, 5, 2), (2, 1, 9, 4), (1, 3, 9, 4)])
@pytest.mark.parametrize("shared", [False, True])
def test_copies(dev, layers, heads, pages, n, shared):
    pools = pools_of(dev, layers, pages, heads)
    order = np.random.default_rng(n).permutation(pages).astype(np.int32)
    dst, src = order[:n], order[n:2 * n]
    if shared:
        src = np.resize(src[:(n + 2) // 3], n)
    want = [p.clone() for p in pools]
    s, d = (torch.from_numpy(x.astype(np.int64)).to(dev) for x in (src, dst))
    for w in want:
        w.view(torch.int16).index_copy_(0, d, w.view(torch.int16).index_select(0, s))
    kernels.kv_copy_pages(pools, src, dst)
    torch.cuda.synchronize()
    assert all(same(p, w) for p, w in zip(pools, want))


def test_pages_past_32_bits_of_elements(dev):
    n = 2**31 // (2 * 4 * 1024) + 5
    pool = torch.empty(n, 2, 4, 1024, dtype=torch.bfloat16, device=dev)
    pool[:4].normal_()
    pool[-3:].normal_()
    want = pool[0].clone(), pool[-1].clone()
    kernels.kv_copy_pages([pool], [0, n - 1], [n - 2, 2])
    assert same(pool[n - 2], want[0]) and same(pool[2], want[1])
    assert same(pool[0], want[0]) and same(pool[-1], want[1])


def test_no_pairs(dev):
    pools = pools_of(dev, 1, 3, 4)
    want = pools[0].clone()
    kernels.kv_copy_pages(pools, [], [])
    assert same(pools[0], want)


def test_captured_copy_keeps_its_pairs(dev):
    """The ids are read when the call is made: a graph holds them although the caller's array changes."""
    pools = pools_of(dev, 3, 10, 8)
    src, dst = np.array([1, 2], dtype=np.int32), np.array([5, 6], dtype=np.int32)
    kernels.kv_copy_pages(pools, src, dst)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kernels.kv_copy_pages(pools, src, dst)
    src[:], dst[:] = 3, 4
    for seed in range(3):
        for p, q in zip(pools, pools_of(dev, 3, 10, 8, seed + 1)):
            p.copy_(q)
        want = [p.clone() for p in pools]
        for w in want:
            w[5], w[6] = w[1], w[2]
        g.replay()
        torch.cuda.synchronize()
        assert all(same(p, w) for p, w in zip(pools, want))


@pytest.mark.parametrize("change,msg", [
    (dict(src=[1], dst=[10]), "outside the pool"), (dict(src=[1, 2], dst=[3, 3]), "two pairs"),
    (dict(src=[1, 2], dst=[2, 3]), "source and a destination"), (dict(src=[1, 2], dst=[3]), "same length"),
    (dict(src=lambda dev: torch.tensor([1], device=dev)), "host integers"), (dict(pools=[]), "no pools"),
    (dict(pools=lambda dev: [torch.zeros(10, 2, 4, 1024, device=dev)]), "torch.bfloat16"),
    (dict(pools=lambda dev: pools_of(dev, 1, 10, 4) + pools_of(dev, 1, 9, 4)), "same shape"),
    (dict(pools=lambda dev: [p.cpu() for p in pools_of(dev, 1, 10, 4)]), "GPU tensor"),
])
def test_refusals(dev, change, msg):
    args = dict(pools=pools_of(dev, 2, 10, 4), src=[1], dst=[2])
    args.update({k: v(dev) if callable(v) else v for k, v in change.items()})
    with pytest.raises(ValueError, match=msg):
        kernels.kv_copy_pages(**args)


@pytest.mark.parametrize("seed", range(3))
def test_shared_cache_random_use(dev, seed):
    play(dev, seed, 40)


def test_static_rows_copy_as_before(dev):
    kv = PagedKV(n_layers=3, n_rows=4, pages_per_row=7, n_heads=16, device=dev, shuffle_seed=1)
    for p in kv.pools:
        p.normal_()
    want = [p.clone() for p in kv.pools]
    kv.copy_row_pages(0, 3, 100)
    for p, w in zip(kv.pools, want):
        w[kv.table_host[3]] = w[kv.table_host[0]]
        assert same(p, w)


def test_a_replaced_pool_is_checked_again(dev):
    kv = PagedKV(n_layers=2, n_rows=2, pages_per_row=4, n_heads=4, device=dev)
    kv.copy_row_pages(0, 1, 20)
    kv.pools[0] = kv.pools[0][:6]  # the same address, fewer pages
    with pytest.raises(ValueError, match="same shape"):
        kv.copy_row_pages(0, 1, 20)


def test_long_use_keeps_to_its_window_of_pages(dev):
    """One row written and released behind its window: the pool never holds more than the window needs."""
    kv = SharedPagedKV(n_layers=1, n_rows=1, pages_per_row=40, n_heads=4, device=dev, n_pages=8)
    m = Model(kv)
    for pos in range(0, 600, 10):
        m.release_before(0, pos - 64, 16)
        m.write(0, pos, pos + 10)
    m.check()
