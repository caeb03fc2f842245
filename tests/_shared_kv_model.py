"""A plain model of rows that share pages, to hold SharedPagedKV against (no tests here)."""

import random

import torch

from yapd_amd.paged import PAGE_SIZE, SharedPagedKV


class Model:
    """Every row as a list of tags, one per position (None: not mapped or never written).  A tag is written
    into the first element of the position's K in head 0 of every layer's pool, plus the layer."""

    def __init__(self, kv: SharedPagedKV):
        self.kv = kv
        self.rows = [[None] * (kv.pages_per_row * PAGE_SIZE) for _ in range(kv.n_rows)]
        self.next_tag = 1

    def write(self, row, begin, end):
        self.kv.reserve(row, begin, end)
        for pos in range(begin, end):
            page = int(self.kv.table_host[row, pos // PAGE_SIZE])
            assert page > 0 and self.kv.refcount(page) == 1
            tag = self.next_tag = self.next_tag % 250 + 1
            for li, pool in enumerate(self.kv.pools):
                pool[page, 0, 0, (pos % PAGE_SIZE) * 64] = (tag + li) % 251
            self.rows[row][pos] = tag

    def fork(self, src, dst, n):
        self.kv.fork(src, dst, n)
        whole = n if n % PAGE_SIZE == 0 else (n // PAGE_SIZE + 1) * PAGE_SIZE  # the last page's slots come along
        for r in dst:
            self.rows[r] = self.rows[src][:whole] + [None] * (len(self.rows[src]) - whole)

    def release(self, row):
        self.kv.release(row)
        self.rows[row] = [None] * len(self.rows[row])

    def release_before(self, row, position, sinks):
        self.kv.release_before(row, position, sinks)
        for c in range(self.kv.pages_per_row):
            if c * PAGE_SIZE >= sinks and (c + 1) * PAGE_SIZE <= position:
                self.rows[row][c * PAGE_SIZE:(c + 1) * PAGE_SIZE] = [None] * PAGE_SIZE

    def check(self):
        kv = self.kv
        table = kv.table.cpu()
        assert table.tolist() == kv.table_host.tolist()
        pools = [p.cpu() for p in kv.pools]
        for r, tags in enumerate(self.rows):
            for pos, tag in enumerate(tags):
                if tag is not None:
                    page = int(table[r, pos // PAGE_SIZE])
                    assert page > 0
                    for li, pool in enumerate(pools):
                        assert float(pool[page, 0, 0, (pos % PAGE_SIZE) * 64]) == (tag + li) % 251, (r, pos, li)
        uses = {}
        for page in kv.table_host.ravel().tolist():
            if page:
                uses[page] = uses.get(page, 0) + 1
        for page in range(1, kv.n_pages):
            assert kv.refcount(page) == uses.get(page, 0)
        assert kv.free_pages == kv.n_pages - 1 - len(uses)


def play(device, seed, steps, pages=60):
    """Random use of a small cache; every step is checked."""
    rng = random.Random(seed)
    kv = SharedPagedKV(n_layers=2, n_rows=5, pages_per_row=6, n_heads=4, device=device, n_pages=pages)
    m = Model(kv)
    for _ in range(steps):
        op = rng.choice(["write", "write", "fork", "release", "before", "compact", "swap"])
        r = rng.randrange(kv.n_rows)
        try:
            if op == "write":
                a = rng.randrange(90)
                m.write(r, a, a + rng.randint(0, min(96 - a, 40)))
            elif op == "fork":
                dst = rng.sample([x for x in range(kv.n_rows) if x != r], rng.randint(1, 3))
                for d in dst:
                    m.release(d)
                m.fork(r, dst, rng.randint(0, 96))
            elif op == "release":
                m.release(r)
            elif op == "before":
                m.release_before(r, rng.randint(-5, 100), rng.choice([0, 5, 16, 20]))
            elif op == "compact":
                n = kv.compact()
                assert kv.table_host.max() < n == kv.n_pages - kv.free_pages
            else:
                o = rng.randrange(kv.n_rows)
                kv.swap_rows(r, o)
                m.rows[r], m.rows[o] = m.rows[o], m.rows[r]
        except RuntimeError as e:
            assert "out of pages" in str(e)
        m.check()
