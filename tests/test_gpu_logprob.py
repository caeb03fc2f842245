"""GPU: token log probabilities, entropy and top alternatives against 64 bits; tokens of the top exactly."""

import math

import pytest
import torch

from oracle import logprob as OL
from yapd_amd import kernels, scoring

pytestmark = pytest.mark.gpu
INF = math.inf


def check(logits, tokens, k, res):
    n = logits.reshape(-1, logits.shape[-1])
    lp, ent, top_lp, top = OL.token_logprobs(n, tokens.reshape(-1), k)
    tol, tol_e = OL.tolerances(n, ent)
    torch.cuda.synchronize()

    def near(got, want, tol):
        got = got.cpu().double().reshape(want.shape)
        same = (got == want) | (got.isnan() & want.isnan())
        bad = ~(same | ((got - want).abs() <= tol + 2.0 ** -24 * want.abs()))
        assert not bool(bad.any()), (bad.nonzero()[0].tolist(), got[bad][0].item(), want[bad][0].item())
    near(res.logprob, lp, tol)
    near(res.entropy, ent, tol_e)
    if k:
        assert torch.equal(res.top_token.cpu().reshape(top.shape), top)
        near(res.top_logprob, top_lp, tol[:, None])
    else:
        assert res.top_logprob is None and res.top_token is None


def rows(n, V, dtype, seed, std=3.0):
    g = torch.Generator().manual_seed(seed)
    return (std * torch.randn(n, V, generator=g)).to(dtype), torch.randint(0, V, (n,), generator=g)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 63, 64, 130, 257, 520, 2047, 2048, 8192, 8194, 10241, 20500, 65537, 100003])
def test_vocabularies(dev, V, dtype):
    for k in (0, 1, 3, 20, 32):
        if k > V:
            continue
        x, t = rows(3, V, dtype, V + k)
        check(x, t, k, scoring.token_logprobs(x.to(dev), t.to(dev), k))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [1, 2, 65, 300, 2100])
def test_row_counts(dev, n, dtype):
    x, t = rows(n, 1001, dtype, n)
    check(x, t, 5, scoring.token_logprobs(x.to(dev), t.to(dev), 5))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("offset", range(9))
def test_any_alignment_and_pitch(dev, offset, dtype):
    """Rows that start at any element of a granule, in a wider buffer of NaN."""
    rws, bl, V, pitch = 3, 4, 1003, 1003 + offset
    x, t = rows(rws * bl, V, dtype, offset)
    buf = torch.full((rws, bl * pitch + 24 + offset), math.nan, dtype=dtype, device=dev)
    view = buf[:, offset:offset + bl * pitch].unflatten(1, (bl, pitch))[..., :V]
    view.copy_(x.view(rws, bl, V))
    check(x, t, 4, scoring.token_logprobs(view, t.view(rws, bl).to(dev), 4))


def special(V, dtype):
    """Rows that go wrong easily, and what they are."""
    lo, hi = torch.finfo(dtype).min, torch.finfo(dtype).max
    base = rows(1, V, dtype, 7)[0][0]
    out = {"constant": torch.full((V,), 2.5), "zeros of both signs": torch.zeros(V) * torch.where(torch.arange(V) % 3 == 0, -1., 1.),
           "rising": torch.linspace(-20, 20, V), "falling": torch.linspace(20, -20, V),
           "all lowest": torch.full((V,), lo), "all largest": torch.full((V,), hi), "all -inf": torch.full((V,), -INF),
           "all NaN": torch.full((V,), math.nan), "tiny": torch.full((V,), 1e-38)}
    for name, at, value in [("one -inf", [0], -INF), ("last -inf", [V - 1], -INF), ("a NaN", [V // 2], math.nan),
                            ("+inf", [V // 3], INF), ("two +inf", [1, V - 2], INF), ("far above", [V // 2], 1e30)]:
        out[name] = base.float().clone()
        out[name][at] = value
    for name, keep in (("one allowed", [V // 2]), ("three allowed", [3, V // 2, V - 1])):
        for fill, what in ((-INF, "-inf"), (lo, "lowest")):
            r = torch.full((V,), fill)
            r[keep] = base.float()[keep]
            out[f"{name}, rest {what}"] = r
    few = torch.full((V,), -5.0)
    few[::max(1, V // 40)] = 3.0  # 40 equal best
    out["equal best"] = few
    block = torch.full((V,), -9.0)
    block[V // 2:V // 2 + 50] = torch.linspace(1, 2, min(50, V - V // 2))  # the best next to each other
    out["best in one place"] = block
    out["best before a signalling NaN"] = base.float().clone()
    out["best before a signalling NaN"][:64] = 50.0 + torch.arange(64) / 4
    x = torch.stack([r.to(dtype) for r in out.values()])
    bits, snan = (torch.int16, 0x7f81) if dtype == torch.bfloat16 else (torch.int32, 0x7f800001)
    x[-1].view(bits)[1::2] = snan  # not by value: a conversion would quiet it
    return list(out), x


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [100, 8194, 50001])
@pytest.mark.parametrize("k", [0, 1, 5, 32])
def test_special_rows(dev, V, k, dtype):
    names, x = special(V, dtype)
    t = torch.full((len(names),), V // 2)
    res = scoring.token_logprobs(x.to(dev), t.to(dev), k)
    for i, name in enumerate(names):
        one = scoring.TokenLogprobs(*(None if v is None else v[i:i + 1] for v in vars(res).values()))
        try:
            check(x[i:i + 1], t[i:i + 1], k, one)
        except AssertionError as e:
            raise AssertionError(f"{name}: {e}") from e


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [1400, 4001, 8194, 20500])
@pytest.mark.parametrize("k", [0, 4, 32])
def test_special_rows_among_many(dev, V, k, dtype):
    """2048 rows or more: one wave each."""
    names, x = special(V, dtype)
    t = torch.full((len(names),), V // 2)
    times = 2048 // len(names) + 1
    res = scoring.token_logprobs(x.to(dev).repeat(times, 1), t.to(dev).repeat(times), k)
    for first in (0, len(names), (times - 1) * len(names)):  # rows of other alignments where V is odd
        for i, name in enumerate(names):
            at = slice(first + i, first + i + 1)
            one = scoring.TokenLogprobs(*(None if v is None else v[at] for v in vars(res).values()))
            try:
                check(x[i:i + 1], t[i:i + 1], k, one)
            except AssertionError as e:
                raise AssertionError(f"{name} at row {first + i}: {e}") from e


def test_tokens_outside_the_vocabulary(dev):
    x, t = rows(5, 500, torch.bfloat16, 0)
    t = torch.tensor([-1, -100, 499, 500, 2**40])
    res = scoring.token_logprobs(x.to(dev), t.to(dev), 2)
    check(x, t, 2, res)
    assert res.logprob[:2].tolist() == [0.0, 0.0] and bool(res.logprob[3:].isnan().all())


def test_same_bits_twice_and_under_capture(dev):
    x, t = rows(200, 8194, torch.bfloat16, 3)
    x, t = x.to(dev), t.to(dev)
    first = scoring.token_logprobs(x, t, 8)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        res = scoring.token_logprobs(x, t, 8)
    for seed in (3, 4, 5):
        y, u = rows(200, 8194, torch.bfloat16, seed)
        x.copy_(y)
        t.copy_(u)
        g.replay()
        eager = scoring.token_logprobs(x, t, 8)
        torch.cuda.synchronize()
        for a, b in zip(vars(res).values(), vars(eager).values()):
            assert torch.equal(a, b)
        check(y, u, 8, res)
        if seed == 3:
            assert all(torch.equal(a, b) for a, b in zip(vars(res).values(), vars(first).values()))


@pytest.mark.parametrize("dtype,V", [(torch.float32, 147457), (torch.float32, 500009), (torch.bfloat16, 294913),
                                     (torch.bfloat16, 1000003)])
def test_vocabularies_whose_maxima_are_of_more_than_three_granules(dev, dtype, V):
    x, tokens = rows(3, V, dtype, V)
    x[1] = -math.inf
    x[1, 5::1000] = 1.0
    check(x.to(dev), tokens.to(dev), 32, scoring.token_logprobs(x.to(dev), tokens.to(dev), top_k=32))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_past_32_bits_of_elements(dev, dtype):
    x, _ = rows(3, 1000, dtype, 5)
    far = torch.empty(2**31 + 4096, dtype=dtype, device=dev).as_strided((3, 1000), (2**30 + 1024, 1))
    far.copy_(x)
    tokens = torch.tensor([0, 999, 500], device=dev)
    check(far, tokens, 8, scoring.token_logprobs(far, tokens, top_k=8))


def test_empty(dev):
    res = scoring.token_logprobs(torch.empty(0, 50, dtype=torch.bfloat16, device=dev),
                                 torch.empty(0, dtype=torch.int64, device=dev), 3)
    assert res.logprob.shape == (0,) and res.top_token.shape == (0, 3)


@pytest.mark.parametrize("change,msg", [
    (dict(top_k=33), "top_k"), (dict(top_k=-1), "top_k"), (dict(top_k=21), "top_k"),
    (dict(logits=lambda x: x.half()), "logits must be torch.bfloat16"), (dict(logits=lambda x: x.t()), "unit last stride"),
    (dict(logits=lambda x: x[0]), "logits must be"), (dict(tokens=lambda t: t.int()), "tokens must be torch.int64"),
    (dict(tokens=lambda t: t[:2]), "leading shape"), (dict(tokens=lambda t: t.cpu()), "GPU tensor"),
])
def test_refusals(dev, change, msg):
    x, t = rows(4, 20, torch.bfloat16, 0)
    args = dict(logits=x.to(dev), tokens=t.to(dev), top_k=2)
    args.update({k: v(args[k]) if callable(v) else v for k, v in change.items()})
    with pytest.raises(ValueError, match=msg):
        scoring.token_logprobs(**args)
