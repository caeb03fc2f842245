"""GPU: token log probabilities that are infinite or none: -inf logits among finite ones have exactly -inf, whether they are
the given token or among the alternatives; a row with NaN or +inf has NaN.  Infinities are compared as they are."""

import math

import pytest
import torch

from oracle import logprob as OL
from tests.test_gpu_logprob import special
from yapd_amd import scoring

pytestmark = pytest.mark.gpu


def near(got, want, tol):
    """Finite values within ``tol`` of finite ones; NaN for NaN, an infinity for the same one."""
    got = got.cpu().double().reshape(want.shape)
    same = (got == want) | (got.isnan() & want.isnan())
    close = got.isfinite() & want.isfinite() & ((got - want).abs() <= tol + 2.0 ** -24 * want.abs())
    bad = ~(same | close)
    assert not bool(bad.any()), (bad.nonzero()[0].tolist(), got[bad][0].item(), want[bad][0].item())


def check(x, tokens, k, res, names):
    lp, ent, top_lp, top = OL.token_logprobs(x, tokens, k)
    tol, tol_e = OL.tolerances(x, ent)
    for i, name in enumerate(names):
        try:
            near(res.logprob[i], lp[i], tol[i])
            near(res.entropy[i], ent[i], tol_e[i])
            if k:
                assert torch.equal(res.top_token[i].cpu(), top[i])
                near(res.top_logprob[i], top_lp[i], tol[i])
        except AssertionError as e:
            raise AssertionError(f"{name}: {e}") from e


# rows a call: special()'s 22, of eight waves each from V = 4001 on, or 90 times as many, of one wave
@pytest.mark.parametrize("times", [1, 90])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [100, 4001, 8194, 20500])
def test_special_rows(dev, V, dtype, times):
    names, x = special(V, dtype)
    for k in (0, 1, 5, 32):
        # the token: one that is kept, the first (masked in some rows), the last (-inf in one)
        for token in (V // 2, 0, V - 1, 5):
            t = torch.full((len(names),), token)
            res = scoring.token_logprobs(x.to(dev).repeat(times, 1), t.to(dev).repeat(times), k)
            for first in {0, (times - 1) * len(names)}:
                part = scoring.TokenLogprobs(*(None if v is None else v[first:first + len(names)] for v in vars(res).values()))
                check(x, t, k, part, names)


@pytest.mark.parametrize("n", [4, 1600])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [40, 300, 2500, 8194, 17000])
def test_masked_tokens(dev, V, dtype, n):
    """A token of probability 0 beside finite ones: -inf exactly; alternatives past the allowed ones: -inf, lowest index first."""
    g = torch.Generator().manual_seed(V)
    x = (3 * torch.randn(4, V, generator=g)).to(dtype)
    t = torch.randint(0, V, (4,), generator=g)
    x[0, t[0]] = -math.inf
    x[1] = -math.inf
    x[1, (t[1] + torch.arange(1, 6)) % V] = torch.tensor([0.5, -1.0, 2.0, 2.0, 3.0]).to(dtype)
    x[2, torch.rand(V, generator=g) < 0.5] = -math.inf
    x[2, t[2]], x[2, (t[2] + 1) % V] = -math.inf, 1.0
    res = scoring.token_logprobs(x.repeat(n // 4, 1).to(dev), t.repeat(n // 4).to(dev), 20)
    assert bool((res.logprob.view(-1, 4)[:, :3] == -math.inf).all()) and bool(res.logprob.view(-1, 4)[:, 3].isfinite().all())
    assert bool((res.top_logprob.view(-1, 4, 20)[:, 1, 5:] == -math.inf).all())
    for first in {0, n - 4}:
        part = scoring.TokenLogprobs(*(v[first:first + 4] for v in vars(res).values()))
        check(x, t, 20, part, ["own masked", "five allowed", "half allowed", "plain"])
