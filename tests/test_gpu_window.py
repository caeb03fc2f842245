"""GPU: attention with a sliding window and sinks over the paged cache, against the definition in 64 bits.
Everything that no query sees -- pages behind the window, slots past the end -- holds NaN, and the table entries of
pages that no query sees are out of range, so a key that leaks into a result shows."""

import pytest
import torch

from tests._window_cases import Case
from yapd_amd import kernels

pytestmark = pytest.mark.gpu


# (q per row, kv lengths, heads, window, sinks)
UNIFORM = [
    (1, [1], 4, 1, 0),                               # one key
    (1, [40, 1, 17, 300, 299], 16, 1, 0),            # every query sees itself only
    (1, [40, 33, 17, 300, 301], 16, 16, 4),
    (1, [500, 31, 32, 33, 64, 65, 800], 8, 100, 33),
    (1, [1, 2, 15, 16, 17], 4, 10000, 10000),        # window and sinks past everything
    (1, [700] * 70, 16, 257, 16),                    # enough rows for one wave a head
    (5, [5, 6, 21, 400], 4, 37, 3),
    (16, [16, 100, 333], 16, 64, 0),
    (17, [17, 50, 640], 8, 48, 20),
    (32, [32, 33, 300, 1000], 16, 500, 33),
    (33, [40, 90, 700], 4, 20, 1),                   # window shorter than the block
    (48, [48, 500, 130], 16, 200, 16),
    (64, [64, 65, 1000], 16, 333, 64),
    (64, [2000] * 40, 4, 129, 5),
    (65, [65, 500], 4, 100, 7),                      # more queries than a tile
    (200, [200, 211, 450], 8, 90, 16),
    (300, [300, 1000], 4, 1000, 0),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("q,kv,H,window,sinks", UNIFORM)
def test_uniform_rows(dev, q, kv, H, window, sinks, causal):
    c = Case(q_lens=[q] * len(kv), kv_lens=kv, H=H, window=window, sinks=sinks, causal=causal, seed=q + len(kv))
    c.check(c.run(dev, kernels))


PACKED = [
    ([3], [3], 4, 2, 0),
    ([1, 0, 5, 64, 2], [1, 9, 40, 64, 2], 16, 17, 4),       # a row without queries, one-token rows
    ([0, 0, 70, 0], [0, 5, 100, 0], 4, 33, 3),              # rows without keys
    ([129, 1, 700, 33], [200, 600, 700, 33], 8, 150, 20),
    ([128, 256, 1], [128, 256, 1], 4, 64, 0),
    ([500, 40], [1500, 2000], 16, 257, 31),
    ([7] * 100, [7 + 3 * i for i in range(100)], 4, 50, 5),  # more rows than one step of the row search
    ([1, 900], [5000, 900], 4, 4000, 64),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("q,kv,H,window,sinks", PACKED)
def test_packed_rows(dev, q, kv, H, window, sinks, causal):
    c = Case(q_lens=q, kv_lens=kv, H=H, window=window, sinks=sinks, causal=causal, seed=len(q), packed=True, tail_q=5)
    c.check(c.run(dev, kernels))
    c.check(c.run(dev, kernels, max_q=max(q), max_kv=max(kv)))


@pytest.mark.parametrize("rows,H", [(2, 4), (63, 4), (64, 4), (65, 4), (64, 16), (44, 64)])
@pytest.mark.parametrize("window,causal", [(1, True), (200, True), (200, False), (100000, True)])
def test_packed_prompts_among_short_rows(dev, rows, H, window, causal):
    """Rows of 0 to 3 tiles of 128 queries behind 0 to 3 tiles of earlier keys, some of them empty; of few and of many
    workgroups."""
    g = torch.Generator().manual_seed(rows + H)
    q = [int(x) for x in torch.tensor([0, 1, 2, 70, 127, 128, 129, 300])[torch.randint(0, 8, (rows,), generator=g)]]
    q[-1] = 131
    past = [int(x) for x in torch.randint(0, 400, (rows,), generator=g)]
    past[0] = 0
    if rows > 40:  # the oracle's time
        q = [min(x, 131) for x in q]
    c = Case(q_lens=q, kv_lens=[a + b for a, b in zip(q, past)], H=H, window=window, sinks=3, causal=causal, packed=True,
             tail_q=3)
    c.check(c.run(dev, kernels))


def test_packed_many_rows(dev):
    """More rows than 64 * 64: three steps of the row search."""
    n = 4500
    c = Case(q_lens=[1 + i % 3 for i in range(n)], kv_lens=[1 + i % 3 + i % 40 for i in range(n)], H=4, window=9,
             sinks=2, causal=True, packed=True, tail_q=1)
    c.check(c.run(dev, kernels, max_q=3))


@pytest.mark.parametrize("rows,H,bl,kv,window", [(1, 4, 1, 30000, 30000), (1, 16, 1, 9000, 6000), (2, 4, 16, 20000, 15000),
                                                 (1, 4, 40, 12000, 12000), (3, 8, 64, 9000, 8000), (1, 4, 150, 9000, 8000)])
def test_split_over_the_keys(dev, rows, H, bl, kv, window):
    c = Case(q_lens=[bl] * rows, kv_lens=[kv - 37 * r for r in range(rows)], H=H, window=window, sinks=20, causal=True,
             seed=kv)
    lib = kernels.load_library()
    assert lib.yapd_attn_window_workspace(rows, bl, rows * bl, 0, H, window, 20, kv) > 0
    out = c.run(dev, kernels)
    c.check(out)
    assert torch.equal(out, c.run(dev, kernels))  # no atomics: the same bits again


def test_split_parts_without_keys(dev):
    """A table that maps far more than the rows hold: most parts are empty."""
    c = Case(q_lens=[1, 3], kv_lens=[5, 40], H=4, window=20000, sinks=4, causal=True, packed=True, extra_cols=2000)
    assert kernels.load_library().yapd_attn_window_workspace(2, 4, 4, 1, 4, 20000, 4, 2000 * 16) > 0
    c.check(c.run(dev, kernels))


def test_strided_queries_and_table(dev):
    """Queries read out of a fused QKV buffer, a table that is a slice of a wider one."""
    c = Case(q_lens=[8] * 4, kv_lens=[8, 100, 57, 333], H=16, window=64, sinks=8, causal=False)
    t = c.device(dev)
    fused = torch.full((4, 8, 3 * 16 * 64), float("nan"), dtype=torch.bfloat16, device=dev)
    q = fused[..., 1024:2048].view(4, 8, 16, 64)
    q.copy_(t["q"])
    wide = torch.full((4, t["table"].shape[1] + 9), -1, dtype=torch.int32, device=dev)
    wide[:, 2:2 + t["table"].shape[1]] = t["table"]
    out = torch.empty(4, 8, 16, 64, dtype=torch.bfloat16, device=dev)
    kernels.attn_window(q, t["pool"], wide[:, 2:2 + t["table"].shape[1]], t["kv_len"], out, 0.125, window=64, sinks=8,
                        causal=False)
    c.check(out)


def test_device_lengths_past_the_table_or_negative(dev):
    """kv_len beyond what the table maps is cut to it; a negative one is an empty row: zeros."""
    c = Case(q_lens=[1, 1, 1], kv_lens=[64, 64, 64], H=4, window=20, sinks=2, causal=True, extra_cols=0)
    t = c.device(dev)
    t["kv_len"].copy_(torch.tensor([64, 2**31 - 1, -3], dtype=torch.int32))
    out = torch.empty_like(t["q"])
    kernels.attn_window(t["q"], t["pool"], t["table"], t["kv_len"], out, 0.125, window=20, sinks=2)
    out = out.cpu().double().view(3, 4, 64)
    assert bool(((out[:2] - c.ref[:2]).abs() <= c.tol[:2]).all()) and bool((out[2] == 0).all())


def test_captured_call_follows_the_device_lengths(dev):
    """One graph, replayed over growing rows with eager work between, each replay against an eager call."""
    H, rows, window, sinks = 8, 3, 100, 10
    c = Case(q_lens=[4] * rows, kv_lens=[900, 500, 700], H=H, window=2000, sinks=sinks, causal=True)  # all keys valid
    t = c.device(dev)
    out = torch.zeros_like(t["q"])
    call = lambda o: kernels.attn_window(t["q"], t["pool"], t["table"], t["kv_len"], o, 0.125, window=window,  # noqa: E731
                                         sinks=sinks)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call(out)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(out)
    for lens in ([4, 4, 4], [100, 33, 64], [900, 500, 700], [5, 500, 699]):
        t["kv_len"].copy_(torch.tensor(lens, dtype=torch.int32))
        g.replay()
        ref = torch.empty_like(out)
        call(ref)
        torch.cuda.synchronize()
        assert torch.equal(out, ref)


def test_captured_packed_call_follows_the_device_rows(dev):
    """One graph of packed prompts, replayed over other partitions of its queries: rows come, go and empty."""
    H, n_q = 4, 450
    c = Case(q_lens=[n_q, 0, 0, 0], kv_lens=[700, 700, 700, 700], H=H, window=5000, sinks=0, causal=True, packed=True)
    t = c.device(dev)
    pool = torch.randn(t["pool"].shape, generator=torch.Generator().manual_seed(1)).bfloat16().to(dev)
    table = torch.arange(4 * t["table"].shape[1], dtype=torch.int32, device=dev).view(4, -1) % pool.shape[0]
    q_start, kv_len = t["q_start"], t["kv_len"]
    call = lambda o: kernels.attn_window(t["q"], pool, table, kv_len, o, 0.125, window=90, sinks=3,  # noqa: E731
                                         q_start=q_start)
    out = torch.empty_like(t["q"])
    call(out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(out)
    for starts, lens in (([0, 450, 450, 450, 450], [700, 0, 0, 0]), ([0, 1, 130, 400, 450], [1, 300, 270, 690]),
                         ([0, 0, 0, 0, 3], [0, 0, 5, 3]), ([7, 140, 140, 140, 440], [133, 9, 9, 301])):
        q_start.copy_(torch.tensor(starts, dtype=torch.int32))
        kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        out.fill_(77.0)
        g.replay()
        ref = torch.full_like(out, 77.0)
        call(ref)
        torch.cuda.synchronize()
        assert torch.equal(out, ref)
        assert bool((out[:starts[0]] == 77.0).all()) and bool((out[starts[-1]:] == 77.0).all())
        assert bool(out[starts[0]:starts[-1]].isfinite().all())


def test_two_graphs_with_parts_do_not_share_a_workspace(dev):
    """Captured calls that split over the keys, replayed on two streams at once."""
    cases = [Case(q_lens=[1], kv_lens=[9000 + i], H=4, window=8000, sinks=4, causal=True, seed=i) for i in range(2)]
    ts = [c.device(dev) for c in cases]
    outs = [torch.zeros_like(t["q"]) for t in ts]
    graphs = []
    for c, t, o in zip(cases, ts, outs):
        kernels.attn_window(t["q"], t["pool"], t["table"], t["kv_len"], o, 0.125, window=8000, sinks=4)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kernels.attn_window(t["q"], t["pool"], t["table"], t["kv_len"], o, 0.125, window=8000, sinks=4)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for c, o in zip(cases, outs):
            c.check(o)


def test_runs_on_the_current_stream(dev):
    c = Case(q_lens=[16] * 2, kv_lens=[300, 20], H=16, window=100, sinks=5, causal=True)
    t = c.device(dev)
    out = torch.empty_like(t["q"])
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(2_000_000)
        q = t["q"] * 1  # made behind the sleep: a call on another stream would read it too early
        kernels.attn_window(q, t["pool"], t["table"], t["kv_len"], out, 0.125, window=100, sinks=5)
    s.synchronize()
    c.check(out)


def test_full_window_agrees_with_the_paged_block_attention(dev):
    """window >= kv_len is the framework's block attention: within two roundings of each other."""
    from yapd_amd.paged import AttnPlan
    kv = [700, 64, 333]
    c = Case(q_lens=[32] * 3, kv_lens=kv, H=16, window=10000, sinks=0, causal=False)
    t = c.device(dev)
    t["table"] = t["table"].clamp(0, c.pool.shape[0] - 1)
    other = torch.empty_like(t["q"])
    AttnPlan(kv, 32, 16, dev).run(t["q"], t["pool"], t["table"], other, 0.125)
    out = c.run(dev, kernels)
    c.check(out)
    c.check(other)


@pytest.mark.parametrize("q", [1, 30, 150])
def test_pages_past_32_bits_of_elements(dev, q):
    """The same rows on the first and on the last pages of a pool of 2^31 + 2^19 elements: the same bits."""
    c = Case(q_lens=[q] * 2, kv_lens=[200, 333], H=4, window=100, sinks=7, causal=True)
    t = c.device(dev)
    n_pages, first = 2**31 // (2 * 4 * 1024) + 64, c.pool.shape[0]
    pool = torch.empty(n_pages, 2, 4, 1024, dtype=torch.bfloat16, device=dev)
    pool[:first], pool[-first:] = t["pool"], t["pool"]
    outs = []
    for shift in (0, n_pages - first):
        out = torch.full_like(t["q"], 77.0)
        kernels.attn_window(t["q"], pool, (t["table"] + shift).contiguous(), t["kv_len"], out, 0.125, window=100, sinks=7)
        outs.append(out)
    c.check(outs[0])
    assert bool((outs[0].view(torch.int16) == outs[1].view(torch.int16)).all())


@pytest.mark.parametrize("rows,H,bl,kv", [(2, 4, 1, 700), (1, 4, 1, 20000), (2, 4, 40, 300), (2, 4, 150, 400),
                                          (1, 4, 150, 9000)])
def test_scales_at_the_ends_of_the_range(dev, rows, H, bl, kv):
    """A power of two moved between the queries and the scale changes nothing, bit for bit; with the
    smallest scale every visible key weighs the same."""
    c = Case(q_lens=[bl] * rows, kv_lens=[kv] * rows, H=H, window=kv, sinks=0, causal=True)
    t = c.device(dev)

    def run(q, scale):
        out = torch.empty_like(q)
        kernels.attn_window(q, t["pool"], t["table"], t["kv_len"], out, scale, window=kv)
        return out.view(torch.int16)

    assert bool((run(t["q"], 0.125) == run(t["q"] * 2.0**-100, 0.125 * 2.0**100)).all())
    assert bool((run(t["q"], 1e-30) == run(torch.zeros_like(t["q"]), 0.125)).all())


def test_no_queries_or_rows_is_no_launch(dev):
    pool = torch.zeros(2, 2, 4, 1024, dtype=torch.bfloat16, device=dev)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    q = torch.empty(0, 4, 64, dtype=torch.bfloat16, device=dev)
    kernels.attn_window(q, pool, i32(0, 1).view(1, 2), i32(5), torch.empty_like(q), 0.125, window=4, q_start=i32(0, 0))
    q = torch.empty(0, 3, 4, 64, dtype=torch.bfloat16, device=dev)
    kernels.attn_window(q, pool, i32(0, 1).view(1, 2), i32(5), torch.empty_like(q), 0.125, window=4)


@pytest.mark.parametrize("change,msg", [
    (dict(window=0), "window >= 1"), (dict(sinks=-1), "sinks >= 0"), (dict(max_kv=0), "max_kv"),
    (dict(max_q=3), "max_q is given by q's shape"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(q=lambda t: t["q"].transpose(1, 2).contiguous().transpose(1, 2)), "heads must be packed"),
    (dict(q=lambda t: t["q"].float()), "q must be torch.bfloat16"),
    (dict(q=lambda t: t["q"][:, :, :3].contiguous()), "pool must be"),
    (dict(table=lambda t: t["table"][:1].expand(2, -1)), "rows must not overlap"),
    (dict(table=lambda t: t["table"][:1]), "table must be"),
    (dict(table=lambda t: t["table"].long()), "table must be torch.int32"),
    (dict(kv_len=lambda t: t["kv_len"][:1]), "kv_len must have rows"),
    (dict(kv_len=lambda t: t["kv_len"].cpu()), "GPU tensor"),
    (dict(out=lambda t: torch.empty(2, 4, 4, 64, dtype=torch.bfloat16, device=t["q"].device)), "out must match q"),
    (dict(workspace=lambda t: torch.empty(4, device=t["q"].device, dtype=torch.float64)), "workspace must be"),
])
def test_refusals(dev, change, msg):
    c = Case(q_lens=[2] * 2, kv_lens=[20, 20], H=4, window=8, sinks=1, causal=True)
    t = c.device(dev)
    args = dict(q=t["q"], pool=t["pool"], table=t["table"], kv_len=t["kv_len"], out=torch.empty_like(t["q"]), scale=0.125,
                window=8, sinks=1)
    args.update({k: v(t) if callable(v) else v for k, v in change.items()})
    with pytest.raises(ValueError, match=msg):
        kernels.attn_window(**args)


def test_a_short_workspace_is_refused(dev):
    c = Case(q_lens=[1], kv_lens=[9000], H=4, window=8000, sinks=0, causal=True)
    with pytest.raises(ValueError, match="workspace"):
        c.run(dev, kernels, workspace=torch.empty(100, dtype=torch.float32, device=dev))
