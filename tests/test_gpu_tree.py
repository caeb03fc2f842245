"""GPU: attention for trees of drafted tokens over the paged cache, bf16 and 8-bit, against the definition in 64 bits.
Everything that no node sees -- pages behind the window, slots past the end, nodes of no mask -- holds NaN, and the table
entries of pages that no node sees are out of range, so a key that leaks into a result shows."""

import pytest
import torch

from tests._tree_cases import Case
from yapd_amd import kernels

pytestmark = pytest.mark.gpu

# (nodes per row, kv lengths, heads, window, sinks)
UNIFORM = [
    (1, [1], 4, None, 0),                             # one key
    (1, [2, 15, 16, 17, 63, 64, 65, 300], 4, None, 0),
    (1, [40, 33, 17, 300, 301], 16, 16, 4),
    (1, [500, 31, 32, 33, 64, 65, 800], 8, 100, 33),
    (1, [400] * 70, 16, 257, 16),                     # more pairs than four waves a head take
    (1, [130] * 200, 16, None, 0),                    # ... than two
    (1, [6000, 5000], 4, None, 0),                    # parts
    (3, [3, 4, 20, 150], 4, None, 0),                 # a row of nodes alone
    (15, [15, 16, 100, 333], 16, 64, 0),
    (16, [16, 31, 33, 640], 8, None, 0),
    (17, [17, 50, 640], 8, 48, 20),
    (24, [3000, 24, 2900], 4, 1000, 7),               # parts
    (32, [32, 33, 300, 700], 16, 500, 33),
    (33, [40, 90, 400], 4, 33, 1),                    # the smallest window
    (48, [48, 300, 130], 16, 200, 16),
    (64, [64, 65, 500], 16, None, 0),
    (64, [66, 80, 127, 128, 129], 4, 70, 64),
    (64, [200] * 34, 16, None, 0),
    (64, [90] * 162, 16, None, 0),
    (64, [3000], 4, None, 0),                         # parts, two waves of nodes
]


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("n,kv,H,window,sinks", UNIFORM)
def test_uniform_rows(dev, n, kv, H, window, sinks, bits):
    c = Case(n_nodes=[n] * len(kv), kv_lens=kv, H=H, bits=bits, window=window, sinks=sinks, seed=n + len(kv))
    c.check(c.run(dev, kernels))


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("kind", ["chain", "siblings", "full", "none", "padded"])
@pytest.mark.parametrize("n,kv", [(7, [7, 9, 120]), (40, [40, 45, 200]), (64, [64, 100])])
def test_masks(dev, kind, n, kv, bits):
    """A row of nodes that see nothing gives zeros; a block's bits past its nodes are ignored."""
    c = Case(n_nodes=[n] * len(kv), kv_lens=kv, H=4, bits=bits, kind=kind, seed=n)
    c.check(c.run(dev, kernels))


PACKED = [
    ([3], [3], 4, None, 0),
    ([1, 0, 5, 64, 2], [1, 9, 40, 64, 2], 16, 64, 4),        # a row without nodes, rows of nodes alone
    ([0, 0, 50, 0], [0, 5, 100, 0], 4, None, 0),             # rows without keys
    ([64, 1, 33, 16, 17, 32], [200, 600, 700, 33, 800, 32], 8, 150, 20),
    ([7] * 60, [7 + 3 * i for i in range(60)], 4, None, 0),
    ([1, 40], [4000, 900], 4, None, 0),
    ([1 + 5 * (i % 13) for i in range(45)], [70 + 11 * (i % 17) for i in range(45)], 16, 100, 5),
]


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("n,kv,H,window,sinks", PACKED)
def test_packed_rows(dev, n, kv, H, window, sinks, bits):
    c = Case(n_nodes=n, kv_lens=kv, H=H, bits=bits, window=window, sinks=sinks, seed=len(n), packed=True, tail_q=5)
    c.check(c.run(dev, kernels, max_kv=max(kv)))


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("rows", [130, 256, 257])
def test_many_ragged_rows(dev, rows, bits):
    """More workgroups than the chip holds: up to 256 rows are taken by cost, each once; rows of no nodes or no keys among them."""
    n = [(0, 1, 3, 40, 2, 17)[i * i % 6] for i in range(rows)]
    kv = [n[i] + i * 37 % 190 for i in range(rows)]
    c = Case(n_nodes=n, kv_lens=kv, H=12, bits=bits, window=120, sinks=5, packed=True, tail_q=3, seed=rows)
    c.check(c.run(dev, kernels))
    c = Case(n_nodes=[1] * rows, kv_lens=[1 + i * 61 % 700 for i in range(rows)], H=32, bits=bits, seed=rows)
    c.check(c.run(dev, kernels))


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("max_q", [1, 20, 40])
def test_rows_longer_than_max_q(dev, max_q, bits):
    """The first max_q nodes of a row are computed as the row's first, a row of more nodes than a mask has bits too."""
    c = Case(n_nodes=[50, 3, 90], kv_lens=[120, 80, 300], H=4, bits=bits, packed=True, max_q=max_q, window=64, sinks=3)
    c.check(c.run(dev, kernels))


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("max_q,window", [(4, 4), (20, 20), (20, 45), (40, 41)])
def test_masks_deeper_than_the_window(dev, max_q, window, bits):
    """A row of more than max_q nodes may have masks of more nodes than the window is long: it bounds the context alone."""
    c = Case(n_nodes=[50, 3, 64], kv_lens=[120, 80, 300], H=4, bits=bits, packed=True, max_q=max_q, window=window, sinks=3,
             kind="full")
    c.check(c.run(dev, kernels))


@pytest.mark.parametrize("bits", [16, 8])
def test_lengths_past_the_table(dev, bits):
    """kv_len is held to what the table maps: nodes keep their distance from the end."""
    c = Case(n_nodes=[5], kv_lens=[48], H=4, bits=bits, extra_cols=0)
    t = c.device(dev)
    out = torch.full_like(t["q"], 77.0)
    kernels.attn_tree(t["q"], t["pool"], t["table"], t["kv_len"] + 1000, t["mask"], out, 0.125)
    c.check(out)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("n,kv,window,sinks", [(5, [0, 3, 4, 5], None, 0), (5, [2, 0, 40, 1], 5, 2), (40, [0, 17, 39], 50, 3),
                                               (64, [1, 0], None, 0)])
def test_rows_of_fewer_keys_than_nodes(dev, n, kv, window, sinks, bits):
    """The first nodes then stand before the row's begin: nobody sees them, and a row without keys gives zeros."""
    c = Case(n_nodes=[n] * len(kv), kv_lens=kv, H=4, bits=bits, window=window, sinks=sinks, seed=n)
    c.check(c.run(dev, kernels))


def test_a_slice_of_a_wider_buffer(dev):
    c = Case(n_nodes=[9, 9], kv_lens=[40, 100], H=8, bits=8)
    t = c.device(dev)
    wide = torch.full((18, 3 * 8 * 64), float("nan"), dtype=torch.bfloat16, device=dev)
    wide[:, 512:1024] = t["q"].view(18, 512)
    out = torch.full_like(t["q"], 77.0)
    kernels.attn_tree(wide[:, 512:1024].view(2, 9, 8, 64), t["pool"], t["table"], t["kv_len"], t["mask"], out, 0.125)
    c.check(out)


def test_a_table_of_other_pitch_and_a_given_workspace(dev):
    c = Case(n_nodes=[2], kv_lens=[5000], H=4, bits=16)
    t = c.device(dev)
    table = torch.zeros(1, t["table"].shape[1] + 9, dtype=torch.int32, device=dev)
    table[:, :t["table"].shape[1]] = t["table"]
    cols = t["table"].shape[1]
    need = kernels.load_library().yapd_attn_tree_workspace(1, 2, 2, 4, 2**30, 0, cols * 16, 16)
    assert need > 0
    ws = torch.full((need,), float("nan"), device=dev)
    out = torch.full_like(t["q"], 77.0)
    kernels.attn_tree(t["q"], t["pool"], table[:, :cols], t["kv_len"], t["mask"], out, 0.125, workspace=ws)
    c.check(out)
    with pytest.raises(ValueError, match="workspace"):
        kernels.attn_tree(t["q"], t["pool"], table[:, :cols], t["kv_len"], t["mask"], out, 0.125, workspace=ws[:need - 1])


def test_one_node_is_the_windowed_attention_of_one_query(dev):
    """The next token: the same keys as kernels.attn_window sees, within both roundings."""
    c = Case(n_nodes=[1, 1, 1], kv_lens=[300, 77, 1], H=8, bits=16, window=50, sinks=4)
    t = c.device(dev)
    a, b = torch.empty_like(t["q"]), torch.empty_like(t["q"])
    kernels.attn_tree(t["q"], t["pool"], t["table"], t["kv_len"], t["mask"], a, 0.125, window=50, sinks=4)
    kernels.attn_window(t["q"], t["pool"], t["table"], t["kv_len"], b, 0.125, window=50, sinks=4)
    tol = 2 * c.tol.view(a.shape).to(dev)
    assert bool(((a.double() - b.double()).abs() <= tol).all())


def test_other_rows_do_not_change_a_row(dev):
    """The same call, and a row beside others of the same sizes: the same bits."""
    c = Case(n_nodes=[20, 20, 20], kv_lens=[200, 90, 333], H=4, bits=8)
    a, b = c.run(dev, kernels), c.run(dev, kernels)
    assert torch.equal(a, b)
    c.q[20:] = 1.0
    assert torch.equal(c.run(dev, kernels)[:1], a[:1])


@pytest.mark.parametrize("bits", [16, 8])
def test_captured_call_follows_lengths_and_masks(dev, bits):
    kv = [90, 200, 65]
    cases = [Case(n_nodes=n, kv_lens=kv, H=4, bits=bits, packed=True, seed=s, kind=k, extra_cols=1, tail_q=30 - sum(n))
             for n, s, k in (([5, 9, 16], 1, "tree"), ([16, 1, 3], 2, "chain"), ([0, 16, 14], 3, "padded"))]
    t = cases[0].device(dev)
    out = torch.full_like(t["q"], 77.0)
    pages = max(c.pool.shape[0] for c in cases)
    pool = torch.zeros(pages, *t["pool"].shape[1:], dtype=t["pool"].dtype, device=dev)
    st = torch.cuda.Stream()
    ws = torch.empty(1, device=dev)

    def call():
        kernels.attn_tree(t["q"], pool, t["table"], t["kv_len"], t["mask"], out, 0.125, q_start=t["q_start"], max_q=16,
                          workspace=ws)

    def fill(c):
        n = c.device(dev)
        for k in ("q", "mask", "table", "kv_len", "q_start"):
            t[k].copy_(n[k])
        pool[:c.pool.shape[0]] = n["pool"]
        out.fill_(77.0)

    fill(cases[0])
    with torch.cuda.stream(st):
        call()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=st):
            call()
    for i in (0, 1, 2, 1, 0):
        fill(cases[i])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        cases[i].check(out)


def test_page_offsets_past_32_bits(dev):
    """A page behind 2^32 bytes of an 8-bit pool and 2^32 elements of a bf16 one."""
    H = 16
    for bits, tile, pages in ((8, 1040, 2**32 // (2 * H * 1040) + 50), (16, 1024, 2**32 // (2 * H * 1024) + 50)):
        c = Case(n_nodes=[3], kv_lens=[40], H=H, bits=bits)
        t = c.device(dev)
        pool = torch.empty(pages, 2, H, tile, dtype=t["pool"].dtype, device=dev)
        pool[-t["pool"].shape[0]:] = t["pool"]
        table = t["table"].clone()
        table[:, :3] += pages - t["pool"].shape[0]
        out = torch.full_like(t["q"], 77.0)
        kernels.attn_tree(t["q"], pool, table, t["kv_len"], t["mask"], out, 0.125)
        c.check(out)
        del pool
