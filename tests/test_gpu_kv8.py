"""GPU: the 8-bit cache written and read back, and accepted tokens moved together, bit for bit against the definition."""

import numpy as np
import pytest
import torch

from oracle import kv8 as OK
from yapd_amd import kernels
from yapd_amd.paged import PagedKV, SharedPagedKV

pytestmark = pytest.mark.gpu


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def vectors(g, *shape):
    """bf16 vectors of very different sizes: zeros, tiny ones, the largest, ties between codes, NaN and infinities."""
    x = torch.randn(*shape, 64, generator=g)
    x *= torch.pow(2.0, torch.randint(-20, 20, (*shape, 1), generator=g))
    flat = x.view(-1, 64)
    n = flat.shape[0]
    for i, row in enumerate((torch.zeros(64), torch.full((64,), 2.0 ** -128), torch.arange(64) * 2.0 ** -133,
                             torch.full((64,), 3.3895e38), torch.arange(64) + 0.5, torch.arange(64) * 2 + 129.0,
                             torch.tensor([float("nan")] * 64), torch.tensor([float("inf"), -float("inf")] * 32),
                             torch.tensor([float("nan"), 1.0] * 32))):
        flat[(i * 7) % n] = row
    return x.bfloat16()


def expected(pool, table, k, v, rows, pos):
    """The pool (CPU copy) after tokens t of row rows[t] went to position pos[t]."""
    pool = pool.clone()
    ck, cv = OK.quantise(k), OK.quantise(v)
    for t, (r, p) in enumerate(zip(rows, pos)):
        if not 0 <= p < table.shape[1] * 16:
            continue
        page = int(table[r, p // 16])
        if not 0 <= page < pool.shape[0]:
            continue
        OK.write(pool, page, p % 16, 0, ck[0][t], ck[1][t])
        OK.write(pool, page, p % 16, 1, cv[0][t], cv[1][t])
    return pool


WRITES = [
    # tokens a row (one number: uniform), first positions, heads, columns
    (1, [0], 4, 1),
    (1, [0, 5, 15, 16, 31, 40], 16, 3),
    (2, [15, 0, 14], 4, 2),
    (16, [0, 16, 5], 8, 4),
    (17, [0, 15, 16], 4, 4),
    (64, [3, 0], 16, 6),
    ([3, 0, 40, 1, 16, 0], [0, 7, 9, 31, 32, 0], 4, 4),
    ([100], [13], 8, 8),
    ([1] * 70 + [33] * 70, [i % 17 for i in range(140)], 4, 4),  # more rows than one step of the row search
    (5, [-3, 30, 2**31 - 3, -2**31, 45], 4, 3),                  # positions before the first and behind what is mapped
]


@pytest.mark.parametrize("n,pos0,H,cols", WRITES)
def test_write(dev, n, pos0, H, cols):
    rows = len(pos0)
    packed = isinstance(n, list)
    lens = n if packed else [n] * rows
    total = sum(lens)
    g = torch.Generator().manual_seed(total)
    tail = 3 if packed else 0  # tokens behind the last row
    k, v = vectors(g, total + tail, H), vectors(g, total + tail, H)
    pages = rows * cols + 2
    table = torch.randperm(pages, generator=g)[:rows * cols].view(rows, cols).int()
    if rows > 2:
        table[1, cols - 1] = pages      # outside the pool: left out
        table[2, 0] = -1
    pool = torch.randint(0, 256, (pages, 2, H, 1040), generator=g, dtype=torch.uint8)
    qkv = torch.zeros(total + tail, 3, H, 64, dtype=torch.bfloat16, device=dev)
    qkv[:, 1], qkv[:, 2] = k.to(dev), v.to(dev)
    got = pool.to(dev)
    start = np.concatenate([[0], np.cumsum(lens)])
    kernels.kv8_write(qkv[:, 1], qkv[:, 2], got, table.to(dev), i32(pos0, dev),
                      q_start=i32(start, dev) if packed else None)
    row_of = np.repeat(np.arange(rows), lens)
    pos = [pos0[r] + t - int(start[r]) for t, r in enumerate(row_of)]
    want = expected(pool, table, k[:total], v[:total], row_of, pos)
    got = got.cpu()
    assert torch.equal(got, want), f"{int((got != want).sum())} bytes differ, first at {(got != want).nonzero()[0].tolist()}"


def test_write_nothing(dev):
    pool = torch.full((2, 2, 4, 1040), 7, dtype=torch.uint8, device=dev)
    x = torch.zeros(0, 4, 64, dtype=torch.bfloat16, device=dev)
    kernels.kv8_write(x, x, pool, i32([[0]], dev), i32([0], dev))
    kernels.kv8_write(x, x, pool, i32([[0]], dev), i32([0], dev), q_start=i32([0, 0], dev))
    kernels.kv8_write(x, x, pool, torch.zeros(0, 1, dtype=torch.int32, device=dev), i32([], dev))
    assert bool((pool == 7).all())


@pytest.mark.parametrize("kv,H", [([1], 4), ([16, 17, 0, 100, 33], 16), ([5] * 40, 8)])
def test_unpack(dev, kv, H):
    """Written and read back: the values of the codes, in the bf16 pool's order, whole pages; others stay."""
    g = torch.Generator().manual_seed(len(kv))
    rows, cols = len(kv), max(kv) // 16 + 2
    pages = rows * cols + 1
    t8, t16 = (torch.randperm(pages, generator=g)[:rows * cols].view(rows, cols).int() for _ in range(2))
    pool8 = torch.randint(0, 256, (pages, 2, H, 1040), generator=g, dtype=torch.uint8)
    pool8[..., :1024][pool8[..., :1024] == 128] = 0
    pool8[..., 1024:] = torch.randint(1, 248, (pages, 2, H, 16), generator=g).to(torch.uint8)
    pool = torch.full((pages, 2, H, 1024), 7.0, dtype=torch.bfloat16)
    want = pool.double()
    for r, n in enumerate(kv):
        for c in range((n + 15) // 16):
            for slot in range(16):
                for plane in (0, 1):
                    x = OK.read(pool8, int(t8[r, c]), slot, plane)
                    tile = want[int(t16[r, c]), plane]
                    (tile.view(H, 16, 64)[:, slot] if plane == 0 else tile.view(H, 64, 16)[:, :, slot]).copy_(x)
    for max_kv in (None, max(kv)):
        got = pool.to(dev)
        kernels.kv8_unpack(pool8.to(dev), t8.to(dev), i32(kv, dev), got, t16.to(dev), max_kv=max_kv)
        assert torch.equal(got.cpu().double(), want)


def test_unpack_leaves_out_what_is_not_mapped(dev):
    g = torch.Generator().manual_seed(0)
    pool8 = torch.randint(0, 120, (4, 2, 4, 1040), generator=g, dtype=torch.uint8).to(dev)
    t8 = i32([[0, -1, 2, 9], [1, 2, 3, 0]], dev)
    t16 = i32([[0, 1, -7, 3], [4, 5, 60, 6]], dev)
    pool = torch.full((8, 2, 4, 1024), 7.0, dtype=torch.bfloat16, device=dev)
    kernels.kv8_unpack(pool8, t8, i32([64, 1000], dev), pool, t16)
    touched = [bool((pool[p] != 7).any()) for p in range(8)]
    assert touched == [True, False, False, False, True, True, True, False]
    before = pool.clone()
    kernels.kv8_unpack(pool8, t8, i32([0, -5], dev), pool, t16)
    kernels.kv8_unpack(pool8, t8[:, :2], i32([64, 64], dev), pool[:0 + 8], t16[:, :1], max_kv=5)
    assert torch.equal(pool, before)


def test_gathered_after_reading_back(dev):
    """kv_gather of pages read back gives the codes' values token by token."""
    g = torch.Generator().manual_seed(5)
    n, H = 45, 4
    k, v = vectors(g, n, H), vectors(g, n, H)
    kv = PagedKV(n_layers=1, n_rows=1, pages_per_row=4, n_heads=H, device=dev, shuffle_seed=1, kv_bits=8)
    wide = PagedKV(n_layers=1, n_rows=1, pages_per_row=4, n_heads=H, device=dev, shuffle_seed=2)
    kernels.kv8_write(k.to(dev), v.to(dev), kv.pools[0], kv.table, i32([0], dev))
    kernels.kv8_unpack(kv.pools[0], kv.table, i32([n], dev), wide.pools[0], wide.table)
    ka, va = kernels.kv_gather(wide.pools[0], wide.table[0], n)
    assert torch.equal(ka.cpu().double(), OK.values(*OK.quantise(k)))
    assert torch.equal(va.cpu().double(), OK.values(*OK.quantise(v)))


# --------------------------------------------------------------------------- accepted tokens

KEPT = [
    # (base, kept per row) ...
    ([0], [[0]]),
    ([0], [[3]]),
    ([13, 0, 30], [[0, 2, 5], [], [1]]),
    ([5, 40, 16, 7], [[0, 1, 2, 3], [63], [5, 9, 20, 33, 40, 41, 50, 60], list(range(1, 64))]),
    ([20], [[5, 1, 0, 30, 30, 2]]),                       # any order, twice the same
    ([9], [list(range(63, -1, -1))]),                     # all 64 turned round
    ([50, 2], [[2, 40, -1, 5], [70, 1]]),                 # behind what the row maps, before its first node
]


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("base,kept", KEPT)
def test_keep(dev, base, kept, bits):
    g = torch.Generator().manual_seed(len(base))
    rows, cols, H, layers = len(base), 5, 8, 3
    m = max(max(len(x) for x in kept), 1)
    pages = rows * cols + 1
    table = torch.randperm(pages, generator=g)[:rows * cols].view(rows, cols).int()
    tile = 1024 if bits == 16 else 1040
    pools = [torch.randint(0, 256, (pages, 2, H, tile), generator=g).to(torch.int16 if bits == 16 else torch.uint8)
             for _ in range(layers)]
    want = []
    for p in pools:
        w = p.clone()
        for r, row in enumerate(kept):
            for i, node in enumerate(row):
                a, b = base[r] + node, base[r] + i
                if node < 0 or a >= cols * 16 or b >= cols * 16:
                    continue
                pa, pb = int(table[r, a // 16]), int(table[r, b // 16])
                w[pb, 0, :, b % 16 * 64:b % 16 * 64 + 64] = p[pa, 0, :, a % 16 * 64:a % 16 * 64 + 64]
                w[pb, 1, :, b % 16:1024:16] = p[pa, 1, :, a % 16:1024:16]
                if bits == 8:
                    w[pb, :, :, 1024 + b % 16] = p[pa, :, :, 1024 + a % 16]
        want.append(w)
    idx = torch.full((rows, m + 2), 2**31 - 1, dtype=torch.int32)
    for r, row in enumerate(kept):
        idx[r, :len(row)] = torch.tensor(row, dtype=torch.int32)
    got = [p.to(dev) if bits == 8 else p.to(dev).view(torch.bfloat16) for p in pools]
    kernels.kv_keep(got, table.to(dev), i32(base, dev), idx.to(dev)[:, :m], i32([len(x) for x in kept], dev))
    for a, b in zip(got, want):
        a = a.cpu() if bits == 8 else a.view(torch.int16).cpu()
        assert torch.equal(a, b)


def test_keep_past_32_bits(dev):
    """Pages behind 2^32 elements of the pool."""
    H = 16
    for dtype, tile in ((torch.uint8, 1040), (torch.bfloat16, 1024)):
        n = 2**32 // (2 * H * tile) + 9
        pool = torch.empty(n, 2, H, tile, dtype=dtype, device=dev)
        pool[-2:] = torch.arange(2 * 2 * H * tile, device=dev).remainder(120).to(dtype).view(2, 2, H, tile)
        was = pool[-2:].clone()
        kernels.kv_keep([pool], i32([[n - 1, n - 2]], dev), i32([3], dev), i32([[20]], dev), i32([1], dev))
        want = was.clone()  # position 23 (page n - 2, slot 7) to position 3 (page n - 1, slot 3)
        want[1, 0, :, 192:256] = was[0, 0, :, 448:512]
        want[1, 1, :, 3:1024:16] = was[0, 1, :, 7:1024:16]
        if tile == 1040:
            want[1, :, :, 1024 + 3] = was[0, :, :, 1024 + 7]
        assert torch.equal(pool[-2:], want)
        del pool


def test_keep_many_layers_and_a_captured_call(dev):
    """More layers than one launch; a captured call follows the device's counts."""
    cache = SharedPagedKV(n_layers=70, n_rows=2, pages_per_row=3, n_heads=4, device=dev, n_pages=7, kv_bits=8)
    cache.reserve(0, 0, 40)
    cache.reserve(1, 0, 33)
    g = torch.Generator(device=dev).manual_seed(0)
    fresh = [torch.randint(0, 256, p.shape, generator=g, dtype=torch.uint8, device=dev) for p in cache.pools]
    base, kept, count = i32([10, 3], dev), i32([[0, 4, 9], [2, 3, 7]], dev), i32([0, 0], dev)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=st):
            cache.keep_nodes(base, kept, count)
    for counts in ([3, 0], [0, 3], [2, 9], [1, 1]):
        for p, f in zip(cache.pools, fresh):
            p.copy_(f)
        count.copy_(i32(counts, dev))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for p, f in ((cache.pools[i].cpu(), fresh[i].cpu()) for i in (0, 63, 64, 69)):
            for r, (b, row) in enumerate(((10, [0, 4, 9]), (3, [2, 3, 7]))):
                for i in range(3):
                    src, to = b + (row[i] if i < counts[r] else i), b + i
                    a, c = (int(cache.table_host[r, x // 16]) for x in (src, to))
                    for plane in (0, 1):
                        assert torch.equal(p[c, plane, :, 1024 + to % 16], f[a, plane, :, 1024 + src % 16])
                    assert torch.equal(p[c, 0, :, to % 16 * 64:to % 16 * 64 + 64], f[a, 0, :, src % 16 * 64:src % 16 * 64 + 64])
                    assert torch.equal(p[c, 1, :, to % 16:1024:16], f[a, 1, :, src % 16:1024:16])


def test_copies_of_8_bit_pages(dev):
    pools = [torch.randint(0, 256, (9, 2, 4, 1040), dtype=torch.uint8, device=dev) for _ in range(3)]
    was = [p.clone() for p in pools]
    kernels.kv_copy_pages(pools, [1, 1, 8], [0, 3, 5])
    for p, w in zip(pools, was):
        w[[0, 3, 5]] = w[[1, 1, 8]]
        assert torch.equal(p, w)
    with pytest.raises(ValueError, match="same shape|must be"):
        kernels.kv_copy_pages([pools[0], pools[1].view(torch.int8)], [1], [2])
    with pytest.raises(ValueError):
        kernels.kv_copy_pages([pools[0][..., :1024].contiguous()], [1], [2])


def test_another_stream(dev):
    """Everything on a side stream, behind work that is still running there."""
    g = torch.Generator().manual_seed(2)
    k = vectors(g, 32, 4)
    st = torch.cuda.Stream()
    pool = torch.zeros(4, 2, 4, 1040, dtype=torch.uint8, device=dev)
    x = torch.zeros(32, 4, 64, dtype=torch.bfloat16, device=dev)
    src = k.to(dev)
    table, pos0 = i32([[2, 1]], dev), i32([0], dev)
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        torch.cuda._sleep(2_000_000)
        x.copy_(src)
        kernels.kv8_write(x, x, pool, table, pos0)
    st.synchronize()
    want = expected(torch.zeros(4, 2, 4, 1040, dtype=torch.uint8), torch.tensor([[2, 1]]), k, k, [0] * 32, range(32))
    assert torch.equal(pool.cpu(), want)
