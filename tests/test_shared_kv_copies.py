"""CPU: page copies are refused as on the GPU, and rows copied as pages of their own, among the cache's other uses."""

import random

import numpy as np
import pytest
import torch

from tests._shared_kv_model import Model
from yapd_amd.paged import PAGE_SIZE, PagedKV, SharedPagedKV

CPU = torch.device("cpu")


class CopyModel(Model):
    def copy_row(self, src, dst, n):
        self.kv.copy_row_pages(src, dst, n)
        if src != dst and n:
            whole = -(-n // PAGE_SIZE) * PAGE_SIZE  # the last page's slots come along
            self.rows[dst][:whole] = self.rows[src][:whole]


def play_copies(device, seed, steps, pages=60):
    """Random use with rows copied; every step is checked, and one that finds no page left changes nothing."""
    rng = random.Random(seed)
    kv = SharedPagedKV(n_layers=2, n_rows=5, pages_per_row=6, n_heads=4, device=device, n_pages=pages)
    m = CopyModel(kv)
    for _ in range(steps):
        op = rng.choice(["write", "copy", "copy", "fork", "release", "before", "compact"])
        r, o = rng.randrange(kv.n_rows), rng.randrange(kv.n_rows)
        try:
            if op == "write":
                a = rng.randrange(90)
                m.write(r, a, a + rng.randint(0, min(96 - a, 40)))
            elif op == "copy":
                m.copy_row(r, o, rng.randint(0, 96))
            elif op == "fork" and r != o:
                m.release(o)
                m.fork(r, [o], rng.randint(0, 96))
            elif op == "release":
                m.release(r)
            elif op == "before":
                m.release_before(r, rng.randint(-5, 100), rng.choice([0, 5, 16, 20]))
            else:
                kv.compact()
        except RuntimeError as e:
            assert "out of pages" in str(e)
        m.check()
        for row in kv.table_host:
            mapped = row[row != 0]
            assert len(set(mapped.tolist())) == len(mapped)  # a row maps a page once


@pytest.mark.parametrize("seed,pages", [(0, 60), (1, 60), (2, 60), (3, 12), (4, 20)])
def test_random_use_with_copied_rows(seed, pages):
    play_copies(CPU, seed, 80, pages)


@pytest.mark.gpu
@pytest.mark.parametrize("seed,pages", [(5, 60), (6, 14)])
def test_random_use_with_copied_rows_on_the_gpu(dev, seed, pages):
    play_copies(dev, seed, 40, pages)


def test_a_copied_row_does_not_follow_its_source():
    m = CopyModel(SharedPagedKV(n_layers=1, n_rows=3, pages_per_row=6, n_heads=4, device=CPU, n_pages=40))
    m.write(0, 0, 50)
    m.fork(0, [1], 50)
    m.copy_row(0, 1, 40)   # over pages that it shares with the source
    m.write(0, 0, 96)
    m.copy_row(2, 0, 20)   # from a row that maps nothing: unmapped there too
    m.check()
    assert not m.kv.table_host[0, :2].any() and m.kv.table_host[0, 2:].all()


def test_a_row_is_copied_again_in_a_full_pool():
    """The pages that the destination gives back are enough for its copy."""
    m = CopyModel(SharedPagedKV(n_layers=1, n_rows=3, pages_per_row=4, n_heads=4, device=CPU, n_pages=7))
    m.write(0, 0, 48)
    m.copy_row(0, 1, 48)
    assert m.kv.free_pages == 0
    m.write(0, 0, 20)
    m.copy_row(0, 1, 48)
    m.check()
    m.kv.release(1)
    m.rows[1] = [None] * 64
    m.fork(0, [1], 48)     # shares all: nothing of its own to give back
    m.write(2, 0, 16)
    with pytest.raises(RuntimeError, match="3 needed, 2 free"):
        m.copy_row(0, 1, 48)
    m.check()
    m.copy_row(0, 1, 32)
    m.check()


BAD = [
    ([1], [10], "outside the pool"), ([-1], [2], "page ids"), ([10], [2], "outside the pool"), ([1, 2], [3, 3], "two pairs"),
    ([1, 2], [2, 3], "source and a destination"), ([4], [4], "source and a destination"), ([1, 2], [3], "same length"),
    ([1.0], [2], "page ids"), ([[1]], [[2]], "one-dimensional"),
]


@pytest.mark.parametrize("src,dst,msg", BAD)
def test_copies_are_refused_and_change_nothing(src, dst, msg):
    kv = PagedKV(n_layers=2, n_rows=2, pages_per_row=5, n_heads=4, device=CPU)
    for p in kv.pools:
        p.normal_()
    was = [p.clone() for p in kv.pools]
    with pytest.raises(ValueError, match=msg):
        kv.copy_pages(src, dst)
    assert all(torch.equal(p, w) for p, w in zip(kv.pools, was))


def test_copies_of_a_cpu_cache():
    kv = PagedKV(n_layers=2, n_rows=2, pages_per_row=5, n_heads=4, device=CPU)
    for p in kv.pools:
        p.normal_()
    was = [p.clone() for p in kv.pools]
    kv.copy_pages(np.array([1, 1, 2]), [5, 6, 7])
    kv.copy_pages([], [])
    for p, w in zip(kv.pools, was):
        w[[5, 6, 7]] = w[[1, 1, 2]]
        assert torch.equal(p, w)
