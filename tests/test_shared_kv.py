"""CPU: the shared paged cache against a plain model of its rows, its refusals, and those of the page copy."""

import ctypes

import numpy as np
import pytest
import torch

from tests._shared_kv_model import Model, play
from yapd_amd import kernels
from yapd_amd.paged import PagedKV, SharedPagedKV

CPU = torch.device("cpu")


@pytest.mark.parametrize("seed", range(6))
def test_random_use(seed):
    play(CPU, seed, 60)


def test_random_use_of_a_pool_that_runs_out():
    play(CPU, 100, 120, pages=12)


def make(**kw):
    return SharedPagedKV(**{**dict(n_layers=1, n_rows=4, pages_per_row=5, n_heads=4, device=CPU, n_pages=14), **kw})


def test_fork_shares_whole_pages_and_copies_the_partial_one():
    kv = make()
    m = Model(kv)
    m.write(0, 0, 40)
    m.fork(0, [2, 3], 40)
    t = kv.table_host
    assert t[2, :2].tolist() == t[3, :2].tolist() == t[0, :2].tolist() and len({t[0, 2], t[2, 2], t[3, 2]}) == 3
    assert [kv.refcount(int(p)) for p in t[0, :3]] == [3, 3, 1] and kv.free_pages == 13 - 5
    m.write(2, 35, 50)   # behind the fork: its own pages already
    m.write(3, 0, 1)     # inside a shared page: a copy first
    assert kv.refcount(int(t[0, 0])) == 2
    m.check()


def test_out_of_pages_changes_nothing():
    kv = make(n_pages=4)
    m = Model(kv)
    m.write(0, 0, 33)
    before = kv.table_host.copy()
    with pytest.raises(RuntimeError, match="1 needed, 0 free"):
        kv.fork(0, [1], 33)
    with pytest.raises(RuntimeError, match="out of pages"):
        kv.reserve(1, 0, 80)
    assert (kv.table_host == before).all()
    m.check()
    m.fork(0, [1], 32)
    with pytest.raises(RuntimeError, match="out of pages"):
        kv.reserve(1, 0, 1)  # the shared page would need a copy
    m.check()


def test_copy_row_pages_gives_own_pages():
    kv = make()
    m = Model(kv)
    m.write(0, 0, 30)
    m.fork(0, [1], 32)
    kv.copy_row_pages(0, 1, 30)
    m.rows[1] = list(m.rows[0])
    assert not set(kv.table_host[0, :2]) & set(kv.table_host[1, :2])
    m.check()


def test_static_rows_copy_as_before():
    kv = PagedKV(n_layers=2, n_rows=3, pages_per_row=4, n_heads=4, device=CPU, shuffle_seed=3)
    for p in kv.pools:
        p.normal_()
    was = [p.clone() for p in kv.pools]
    kv.copy_row_pages(0, 2, 40)
    kv.copy_row_pages(1, 1, 40)
    for p, w in zip(kv.pools, was):
        w[kv.table_host[2, :3]] = w[kv.table_host[0, :3]]
        assert torch.equal(p, w)
    kv.table_host[1, :2] = kv.table_host[0, 1:3]  # rows that share pages: read before written
    was = kv.pools[0].clone()
    kv.copy_row_pages(0, 1, 32)
    was[kv.table_host[1, :2]] = was[kv.table_host[0, :2]]
    assert torch.equal(kv.pools[0], was)


@pytest.mark.parametrize("call,msg", [
    (lambda kv: kv.reserve(4, 0, 1), "row 4"), (lambda kv: kv.reserve(0, 0, 81), "positions"),
    (lambda kv: kv.reserve(0, 5, 4), "positions"), (lambda kv: kv.reserve(0, -1, 4), "positions"),
    (lambda kv: kv.fork(0, [1, 1], 4), "distinct"), (lambda kv: kv.fork(0, [0], 4), "distinct"),
    (lambda kv: kv.fork(0, [-1], 4), "row -1"), (lambda kv: kv.fork(0, [1], 81), "n_positions"),
    (lambda kv: kv.fork(1, [0], 16), "map nothing"), (lambda kv: kv.release(9), "row 9"),
    (lambda kv: kv.release_before(9, 4), "row 9"), (lambda kv: kv.release_before(0, 4, -1), "sinks"),
    (lambda kv: kv.copy_row_pages(0, 7, 4), "row 7"), (lambda kv: make(n_pages=1), "two pages"),
])
def test_refusals(call, msg):
    kv = make()
    kv.reserve(0, 0, 20)
    with pytest.raises(ValueError, match=msg):
        call(kv)


# ---- the copy's C entry: refused before any launch

P = 4096
POOLS = (ctypes.c_void_p * 2)(P, 2 * P)


def ints(*v):
    return np.asarray(v, dtype=np.int32)


@pytest.mark.parametrize("pools,layers,pages,heads,src,dst,msg", [
    (None, 2, 8, 4, ints(1), ints(2), b"NULL pointer"), (POOLS, 0, 8, 4, ints(1), ints(2), b"empty shape"),
    (POOLS, 2, 0, 4, ints(1), ints(2), b"n_pages"), (POOLS, 2, 8, 0, ints(1), ints(2), b"empty shape"),
    (POOLS, 2, 8, 4, ints(8), ints(2), b"outside the pool"), (POOLS, 2, 8, 4, ints(1), ints(-1), b"outside the pool"),
    (POOLS, 2, 8, 4, ints(1, 2), ints(3, 3), b"destination of two pairs"),
    (POOLS, 2, 8, 4, ints(1, 3), ints(3, 4), b"source and a destination"),
    (POOLS, 2, 8, 4, ints(5), ints(5), b"source and a destination"),
    ((ctypes.c_void_p * 2)(P, P + 8), 2, 8, 4, ints(1), ints(2), b"16-byte aligned"),
    ((ctypes.c_void_p * 2)(P, None), 2, 8, 4, ints(1), ints(2), b"non-NULL"),
])
def test_c_entry_refuses(pools, layers, pages, heads, src, dst, msg):
    lib = kernels.load_library()
    assert lib.yapd_kv_copy_pages(pools, layers, pages, heads, src.ctypes.data, dst.ctypes.data, len(src), None) == 1
    assert msg in lib.yapd_last_error(), lib.yapd_last_error()


def test_c_entry_without_pairs_launches_nothing():
    assert kernels.load_library().yapd_kv_copy_pages(POOLS, 2, 8, 4, None, None, 0, None) == 0


@pytest.mark.parametrize("ids", [[0.5], [[1]], [-1], [2**31], np.zeros(2, dtype=bool)])
def test_page_ids_are_host_integers(ids):
    with pytest.raises(ValueError):
        kernels.page_ids(ids, "src")


def test_page_ids_of_any_integer_type():
    for ids in ([1, 2], (1, 2), np.array([1, 2], dtype=np.uint8), torch.tensor([1, 2]), np.array([9, 1, 9, 2])[1::2]):
        a = kernels.page_ids(ids, "src")
        assert a.dtype == np.int32 and a.tolist() == [1, 2]
    assert kernels.page_ids([], "src").size == 0
