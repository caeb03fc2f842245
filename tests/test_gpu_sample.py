"""GPU: tokens drawn with given random numbers, against the definition in 64 bits.  A draw that comes within 1e-9 of
another outcome by the oracle's own margin would not be told apart from rounding; no case does unless it says so."""

import math

import pytest
import torch

from oracle import sample as OS
from yapd_amd import kernels, scoring

pytestmark = pytest.mark.gpu


def settings(n, seed):
    g = torch.Generator().manual_seed(seed)
    pick = lambda v, dt: torch.tensor(v, dtype=dt)[torch.randint(0, len(v), (n,), generator=g)]  # noqa: E731
    return dict(u=torch.rand(n, generator=g), T=pick([0.0, 0.3, 0.8, 1.0, 1.0, 1.7, 30.0], torch.float32),
                k=pick([0, 0, 0, 1, 2, 7, 50, 1000, 10**6, -3], torch.int32),
                p=pick([1.0, 1.0, 0.9, 0.95, 0.5, 0.1, 2.0], torch.float32),
                m=pick([0.0, 0.0, 0.02, 0.1, 0.5], torch.float32))


def check(dev, logits, s, min_margin=1e-9):
    """Runs the rows on the GPU and compares; returns the tokens."""
    d = {k: v.to(dev) for k, v in s.items()}
    r = scoring.sample_tokens(logits, d["u"], temperature=d["T"], top_k=d["k"], top_p=d["p"], min_p=d["m"])
    token, logprob, margin = OS.sample_tokens(logits, s["u"], s["T"], s["k"], s["p"], s["m"])
    assert float(margin.min()) >= min_margin, "the case comes too near a border to be decided"
    got, lp = r.token.cpu(), r.logprob.cpu().double()
    assert torch.equal(got, token), f"rows {(got != token).nonzero()[:, 0].tolist()[:9]}: {got[got != token][:9]} for {token[got != token][:9]}"
    nan = logprob.isnan()
    assert torch.equal(lp.isnan(), nan)
    off = (lp - logprob).abs()[~nan]
    assert bool((off <= OS.tolerance(logprob[~nan])).all()), off.max()
    return got


@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 63, 300, 1000, 2047, 8194, 16385, 50001])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("std", [3.0, 0.02])
def test_rows(dev, V, wide, std):
    n = 40 if V < 20000 else 12
    g = torch.Generator().manual_seed(V)
    x = torch.randn(n, V, generator=g) * std
    x = (x if wide else x.bfloat16()).to(dev)
    check(dev, x, settings(n, V + wide))


@pytest.mark.parametrize("n,V", [(600, 300), (530, 2057), (1100, 8194), (300, 12000)])
@pytest.mark.parametrize("wide", [False, True])
def test_many_rows(dev, n, V, wide):
    """More rows than CUs, and than twice as many: other workgroups a row."""
    g = torch.Generator().manual_seed(n)
    x = torch.randn(n, V, generator=g) * torch.tensor([3.0, 0.05, 8.0]).repeat(n)[:n, None]
    x[::7, : V // 3] = -math.inf
    x[3::50] = x[3, 0]
    check(dev, (x if wide else x.bfloat16()).to(dev), settings(n, V), min_margin=0.0)


@pytest.mark.parametrize("V,wide", [(100003, True), (131072, False), (300007, False)])
def test_large_vocabularies(dev, V, wide):
    g = torch.Generator().manual_seed(V)
    x = torch.randn(6, V, generator=g) * 2
    check(dev, (x if wide else x.bfloat16()).to(dev), settings(6, V))


def test_rows_inside_one_granule_at_the_end_of_a_buffer(dev):
    """Rows shorter than 16 bytes at any offset: only granules that hold one of their elements are read."""
    g = torch.Generator().manual_seed(0)
    for wide in (False, True):
        n = 4 if wide else 8
        buf = torch.empty(2**21 // (4 if wide else 2), dtype=torch.float32 if wide else torch.bfloat16, device=dev)
        for off in range(n):
            for V in range(1, n - off + 1):
                x = torch.randn(V, generator=g).to(buf.dtype)
                row = buf[buf.numel() - n + off:][:V].view(1, V)
                row.copy_(x)
                check(dev, row, settings(1, off + V), min_margin=0.0)


def test_strides_and_offsets(dev):
    """Rows that start at any element, a padded pitch, positions of a block."""
    g = torch.Generator().manual_seed(0)
    for wide in (False, True):
        for off in (0, 1, 3, 5):
            buf = torch.full((9, 517), math.nan, dtype=torch.float32 if wide else torch.bfloat16, device=dev)
            x = (torch.randn(9, 500, generator=g) * 2).to(buf.dtype).to(dev)
            buf[:, off:off + 500] = x
            check(dev, buf[:, off:off + 500], settings(9, off))
    x = (torch.randn(3, 5, 1003, generator=g) * 2).bfloat16().to(dev)
    s = settings(15, 1)
    d = {k: v.view(3, 5).to(dev) for k, v in s.items()}
    for view in (x, x.transpose(0, 1).contiguous().transpose(0, 1), x.expand(3, 5, 1003)):
        r = scoring.sample_tokens(view, d["u"], temperature=d["T"], top_k=d["k"], top_p=d["p"], min_p=d["m"])
        token = OS.sample_tokens(x.reshape(15, -1), s["u"], s["T"], s["k"], s["p"], s["m"])[0]
        assert torch.equal(r.token.cpu().view(-1), token)
    one = x[:1, :1].expand(3, 5, 1003)  # the same row everywhere
    r = scoring.sample_tokens(one, d["u"], temperature=0.0)
    assert bool((r.token == one[0, 0].float().argmax()).all())


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("V", [1000, 8194, 40000])
def test_many_equal_logits(dev, V, wide):
    """Rows of one value, of a few values, of a peak over a flat floor: order is by index among equals."""
    g = torch.Generator().manual_seed(V)
    x = torch.zeros(12, V)
    x[1] = -7.5
    x[2] = torch.finfo(torch.bfloat16).min
    x[3:6] = torch.randint(0, 3, (3, V), generator=g).float()
    x[6:9, V // 3] = 4.0
    x[9] = torch.where(torch.rand(V, generator=g) < 0.5, 0.0, -0.0)
    x[10] = torch.arange(V).remainder(5) * 1e-30       # differences far below the bins' width
    x[11, V // 2:] = -math.inf
    x = (x if wide else x.bfloat16()).to(dev)
    s = dict(u=torch.tensor([0.0, 0.37, 0.999, 0.21, 0.83, 0.4, 0.0, 0.123, 0.987, 0.61, 0.77, 0.3]), T=torch.full((12,), 0.9),
             k=torch.tensor([0, 0, 0, 0, 777, 0, 0, 0, 900, 0, 0, 0], dtype=torch.int32),
             p=torch.tensor([1.0, 0.707, 1.0, 0.9, 1.0, 0.31, 1.0, 0.87, 1.0, 1.0, 1.0, 0.9]),
             m=torch.tensor([0.0, 0.0, 0.3, 0.0, 0.0, 0.2, 0.0, 0.0, 0.0, 1.0, 0.0, 0.0]))
    # min-p at exactly a weight and u = 0 are borders that both sides meet exactly
    check(dev, x, s, min_margin=0.0)


def test_equal_logits_one_by_one(dev):
    """V equal logits: token floor(u V), and top-p keeps ceil(p V) of them."""
    V = 4096
    x = torch.full((64, V), 1.5, dtype=torch.bfloat16, device=dev)
    u = torch.arange(64, device=dev) / 64 + 1 / 256
    r = scoring.sample_tokens(x, u, temperature=0.5)
    assert torch.equal(r.token, (u * V).long())
    r = scoring.sample_tokens(x, u, temperature=0.5, top_p=0.25)
    assert torch.equal(r.token, (u * (V // 4)).long())
    r = scoring.sample_tokens(x, u, temperature=0.5, top_k=640)
    assert torch.equal(r.token, (u * 640).long())
    assert bool((r.logprob + math.log(640)).abs().max() < 1e-6)


def test_adversarial_ranges(dev):
    """Values whose bins hold almost everything: a far outlier, clusters, tiny and huge temperatures, subnormals."""
    V = 9000
    g = torch.Generator().manual_seed(4)
    base = torch.randn(V, generator=g)
    rows = [torch.cat([base[:-1] * 1e-6, torch.tensor([-3e38])]), torch.cat([base[:-1] * 1e-3, torch.tensor([30.0])]),
            base * 1e-40, base * 1e30, base * 1e37, base + 1e6, torch.where(base > 0, 5.0, 5.0 + base * 1e-6),
            torch.where(torch.arange(V) % 2 == 0, base * 1e-5, -60.0)]
    x = torch.stack(rows).to(dev)
    for T in (1e-3, 1.0, 1e4):
        for k, p in ((0, 1.0), (300, 0.9), (5000, 0.7), (0, 0.3)):
            s = dict(u=torch.rand(8, generator=g), T=torch.full((8,), T), k=torch.full((8,), k, dtype=torch.int32),
                     p=torch.full((8,), p), m=torch.full((8,), 0.0))
            check(dev, x, s, min_margin=1e-10)


@pytest.mark.parametrize("V", [90, 700, 9000])
def test_bf16_values_of_any_size(dev, V):
    """Rows far outside the usual size of logits: tiny ones and subnormals, huge ones, all below zero, zeros of either
    sign among tiny values, masks of the lowest value; temperatures that leave one token, some, and all."""
    g = torch.Generator().manual_seed(V)
    base = torch.randn(V, generator=g)
    some = torch.rand(V, generator=g) < 0.3
    low = float(torch.finfo(torch.bfloat16).min)
    rows = [base * 1e-4, base * 3e-3, base * 1e-20, base * 1e-39, base * 40, base * 1e4, base * 1e30, base * 1e37,
            -base.abs() - 0.01, -base.abs() * 1e-3, -base.abs() * 100 - 70, -base.abs() * 1e36, base - 100, base + 200,
            torch.where(some, 0.0, base * 1e-4), torch.where(some, -0.0, -base.abs() * 1e-3), torch.where(some, 0.0, -base.abs()),
            torch.where(some, low, base), torch.where(some, low, base * 1e36), torch.where(some, low, -math.inf),
            torch.where(some, 2.0 ** -10, 2.0 ** -11), torch.where(some, 64.0, 63.5), torch.where(some, -64.0, -63.5),
            torch.where(torch.arange(V) == V // 2, 3e38, base), torch.where(some, 1e-4, 20.0)]
    x = torch.stack(rows).bfloat16().to(dev)
    n = len(rows)
    spread = x.cpu().float().where(x.cpu() > -1e30, 0.0).abs().amax(1).clamp_min(1e-38)
    for i, (factor, k, p, m) in enumerate([(1.0, 0, 1.0, 0.0), (0.05, 0, 0.9, 0.0), (0.3, 40, 0.8, 0.1), (1e-4, 0, 1.0, 0.0),
                                           (100.0, 0, 0.97, 0.0), (3.0, V // 2, 1.0, 0.3), (0.0, 0, 1.0, 0.0)]):
        full = lambda v, dt=torch.float32: torch.full((n,), v, dtype=dt)  # noqa: E731
        check(dev, x, dict(u=torch.rand(n, generator=g), T=(spread * factor).clamp_max(1e38), k=full(k, torch.int32), p=full(p),
                           m=full(m)), min_margin=0.0)


def test_rows_without_a_distribution(dev):
    x = torch.randn(6, 8194, device=dev).bfloat16()
    x[0, 8193] = math.nan
    x[1, 5] = math.inf
    x[2] = -math.inf
    x[3] = -math.inf
    x[3, 4711] = -100.0
    x[4, 7] = math.nan
    u = torch.full((6,), 0.99, device=dev)
    for T in (0.0, 1.0):
        r = scoring.sample_tokens(x, u, temperature=T, top_k=50, top_p=0.9, min_p=0.01)
        assert r.token[[0, 1, 2, 4]].tolist() == [-1] * 4 and bool(r.logprob[[0, 1, 2, 4]].isnan().all())
        assert r.token[3] == 4711 and r.logprob[3] == 0.0 and r.token[5] >= 0


def test_numbers_outside_their_range(dev):
    """u below 0, from 1 on or NaN; settings that keep everything or only the first."""
    V = 1000
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(1, V, generator=g) * 2).bfloat16().to(dev)
    order = torch.sort(x[0].float().cpu(), descending=True, stable=True)[1]
    draw = lambda u, **kw: int(scoring.sample_tokens(x, torch.tensor([u], device=dev), **kw).token)  # noqa: E731
    assert draw(-3.0) == order[0] and draw(math.nan) == order[0]
    assert draw(1.0, top_k=20) == order[19] and draw(7.0, top_k=20) == order[19]
    assert draw(0.999, top_p=0.0) == order[0] and draw(0.999, top_p=-1.0) == order[0]
    assert draw(0.999, min_p=1.0) == order[0] and draw(0.999, min_p=5.0) == order[0]
    assert draw(0.999, top_k=1) == order[0] and draw(0.3, temperature=0.0) == order[0]
    assert draw(0.999, top_k=-5) == draw(0.999) == draw(0.999, top_k=10**9, top_p=3.0, min_p=-1.0)
    hot = torch.tensor([math.nan], device=dev)
    assert draw(0.9, temperature=hot) == order[0]
    assert draw(0.25 + 1e-4, temperature=math.inf) == order[250]


def test_numbers_and_tensors_agree(dev):
    x = (torch.randn(33, 8194, device=dev) * 3).bfloat16()
    u = torch.rand(33, device=dev)
    a = scoring.sample_tokens(x, u, temperature=0.8, top_k=40, top_p=0.9, min_p=0.03)
    full = lambda v, dt=torch.float32: torch.full((33,), v, dtype=dt, device=dev)  # noqa: E731
    b = scoring.sample_tokens(x, u, temperature=full(0.8), top_k=full(40, torch.int32), top_p=full(0.9), min_p=full(0.03))
    assert torch.equal(a.token, b.token) and torch.equal(a.logprob, b.logprob)


def test_the_draws_follow_the_distribution(dev):
    """Random numbers at the mid-quantiles: every token is drawn its share of times, to one draw at either end."""
    V, n = 200, 20000
    x = (torch.randn(1, V, generator=torch.Generator().manual_seed(2)) * 1.5).to(dev)
    u = (torch.arange(n, device=dev) + 0.5) / n
    r = scoring.sample_tokens(x.expand(n, V), u, temperature=0.7)
    p = torch.softmax(x[0].double() / 0.7, -1)
    count = torch.bincount(r.token, minlength=V)
    assert bool(((count - p * n).abs() <= 1.01).all())
    assert bool((r.logprob.double() - p.log()[r.token]).abs().max() < 1e-6)


def test_empty_batches(dev):
    r = scoring.sample_tokens(torch.zeros(0, 50, device=dev), torch.zeros(0, device=dev))
    assert r.token.shape == (0,)
    r = scoring.sample_tokens(torch.zeros(4, 0, 50, device=dev), torch.zeros(4, 0, device=dev))
    assert r.logprob.shape == (4, 0)


def test_refusals(dev):
    x, u = torch.zeros(3, 50, device=dev), torch.zeros(3, device=dev)
    for bad in (dict(temperature=-1.0), dict(temperature=math.nan), dict(top_p=math.nan), dict(min_p=math.nan), dict(top_k=1.5),
                dict(temperature=torch.ones(2, device=dev)), dict(top_k=torch.ones(3, device=dev)),
                dict(top_p=torch.ones(3)), dict(min_p=torch.ones(3, 1, device=dev))):
        with pytest.raises(ValueError):
            scoring.sample_tokens(x, u, **bad)
    for logits, uniform in ((x.half(), u), (x.double(), u), (x[0], u), (x, u[:2]), (x, u.double()), (x.t(), torch.zeros(50, device=dev)),
                            (x[:, :0], u), (x, 0.5)):
        with pytest.raises(ValueError):
            scoring.sample_tokens(logits, uniform)
    token, lp = torch.zeros(3, dtype=torch.int32, device=dev), torch.zeros(3, device=dev)
    with pytest.raises(ValueError, match="token"):
        kernels.sample_tokens(x, u, token, lp)


def test_captured_call(dev):
    """A replay draws from what the logits, numbers and settings hold then."""
    x = torch.zeros(20, 8194, dtype=torch.bfloat16, device=dev)
    s = {k: v.to(dev) for k, v in settings(20, 0).items()}
    token, lp = torch.zeros(20, dtype=torch.int64, device=dev), torch.zeros(20, device=dev)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=st):
            kernels.sample_tokens(x, s["u"], token, lp, temperature=s["T"], top_k=s["k"], top_p=s["p"], min_p=s["m"])
    for seed in range(4):
        x.copy_(torch.randn(20, 8194, generator=torch.Generator().manual_seed(seed)) * 3)
        n = settings(20, seed)
        for key in s:
            s[key].copy_(n[key])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = check(dev, x, n)
        assert torch.equal(token.cpu(), want)


@pytest.mark.parametrize("value", [-math.inf, float(torch.finfo(torch.bfloat16).min), -1e4, -100.0])
@pytest.mark.parametrize("n", [300, 700])
def test_rows_masked_for_the_most_part(dev, n, value):
    """Most tokens masked, as -inf, by the lowest value, or by one that a high temperature lets in; rows at any offset."""
    V = 1000
    g = torch.Generator().manual_seed(n)
    x = torch.randn(n, V + 9, generator=g) * 2
    x = x.masked_fill(torch.rand(n, V + 9, generator=g) < 0.9, value).bfloat16().to(dev)
    s = settings(n, 3)
    s["T"] = torch.tensor([0.8, 2.0, 30.0, 1e3]).repeat(n)[:n]
    for off in (0, 1, 4, 9):
        check(dev, x[:, off:off + V], s, min_margin=0.0)


@pytest.mark.parametrize("V", [1003, 9001, 20011])
def test_fp32_rows_of_any_range(dev, V):
    """The least logits at the row's ends, which fill no 16 bytes; ranges past fp32's; temperatures whose bins are wide."""
    g = torch.Generator().manual_seed(V)
    base = torch.randn(V, generator=g)
    ends = base * 0.1
    ends[0], ends[-1] = -15.0, -20.0
    rows = [ends, ends - 1e5, (base * 1.5e38).clamp(-3.3e38, 3.3e38), base * 1e37, base * 1e-37, base * 3e-38,
            torch.where(base > 0, 3e38, -3e38)]
    temps = [5.0, 7.0, 1e38, 1e36, 1e-37, 1e-37, 2e38]
    buf = torch.zeros(len(rows), V + 3, device=dev)
    for off in (0, 1, 3):
        buf[:, off:off + V] = torch.stack(rows).to(dev)
        for k, p, m in ((0, 1.0, 0.0), (0, 0.9, 0.0), (V // 3, 0.8, 0.0), (0, 0.95, 0.01), (0, 1.0, 0.2), (900, 1.0, 0.001)):
            full = lambda v, dt=torch.float32: torch.full((len(rows),), v, dtype=dt)  # noqa: E731
            check(dev, buf[:, off:off + V], dict(u=torch.rand(len(rows), generator=g), T=torch.tensor(temps),
                                                 k=full(k, torch.int32), p=full(p), m=full(m)), min_margin=0.0)


@pytest.mark.parametrize("n", [257, 600, 1025])
def test_many_long_fp32_rows_of_different_settings(dev, n):
    """More rows than CUs with a vocabulary of one row a CU: up to 1024 are taken by what their settings cost, each once."""
    V = 60011
    base = torch.randn(5, V, generator=torch.Generator().manual_seed(n)) * 2
    x = base.to(dev)[torch.arange(n, device=dev) % 5] + torch.arange(n, device=dev)[:, None] / 64
    s = settings(n, n)
    r = scoring.sample_tokens(x, s["u"].to(dev), temperature=s["T"].to(dev), top_k=s["k"].to(dev), top_p=s["p"].to(dev),
                              min_p=s["m"].to(dev))
    for i in range(n):  # a row alone gives the same
        one = {k: v[i:i + 1].to(dev) for k, v in s.items()}
        a = scoring.sample_tokens(x[i:i + 1], one["u"], temperature=one["T"], top_k=one["k"], top_p=one["p"], min_p=one["m"])
        assert torch.equal(a.token, r.token[i:i + 1]) and torch.equal(a.logprob, r.logprob[i:i + 1])
    few = torch.arange(0, n, max(n // 25, 1))
    check(dev, x[few.to(dev)], {k: v[few] for k, v in s.items()}, min_margin=0.0)
