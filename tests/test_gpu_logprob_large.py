"""GPU: token log probabilities of large logits over long rows, whose sums are rescaled many times, against 64 bits."""

import numpy as np
import pytest
import torch

from oracle import logprob as OL
from yapd_amd import scoring

pytestmark = pytest.mark.gpu


def worst_residual(near, steps):
    """The number of ``steps`` significands within a factor of two above ``near`` whose product with log2(e) is rounded the
    most."""
    a = np.float32(2.0 ** np.floor(np.log2(near))) * (1 + np.arange(steps, dtype=np.float32) / steps)
    c = np.float32(1.4426950408889634)
    off = np.abs(np.float64(a * c) - np.float64(a) * np.float64(c))
    return float(a[off.argmax()])


# rows of eight waves (many tiles), of one wave (four tiles, one tile)
SHAPES = [(2, 500009, torch.float32), (2, 1000003, torch.bfloat16), (3, 40000, torch.float32), (1600, 17000, torch.float32),
          (1600, 30000, torch.bfloat16), (1700, 1000, torch.float32)]


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("near", [20, 300, 5000, 40000, 65536, 1e6])
@pytest.mark.parametrize("n,V,dtype", SHAPES)
def test_equal_logits(dev, n, V, dtype, near, sign):
    """A row of one value, and one whose values lie up to 3 below it: maxima that stay from tile to tile, and that move."""
    a = sign * worst_residual(near, 128 if dtype == torch.bfloat16 else 2 ** 16)
    base = torch.full((1, V), a, dtype=torch.float64)
    below = base - 3 * torch.rand(1, V, generator=torch.Generator().manual_seed(V), dtype=torch.float64)
    x = torch.cat([base, below]).to(dtype)
    full = x.repeat((n + 1) // 2, 1)[:n]
    t = torch.arange(n) * 7919 % V
    res = scoring.token_logprobs(full.to(dev), t.to(dev), 4)
    for i in {0, 1, n - 2, n - 1}:
        row = full[i:i + 1]
        lp, ent, top_lp, top = OL.token_logprobs(row, t[i:i + 1], 4)
        tol, tol_e = OL.tolerances(row, ent)
        for got, want, bound in ((res.logprob[i], lp, tol), (res.entropy[i], ent, tol_e), (res.top_logprob[i], top_lp[0], tol)):
            off = (got.cpu().double() - want).abs().max().item()
            assert off <= (bound + 2.0 ** -24 * want.abs().max()).item(), (i, off, bound.item())
        assert torch.equal(res.top_token[i].cpu(), top[0])


@pytest.mark.parametrize("n", [2, 1600])
def test_terms_lost_beside_a_large_one(dev, n):
    """Terms just below half a step of 1: a lane that holds the 1 first adds none of its other V / 64 terms."""
    V = 34800  # 4350 granules: one wave a row from 1536 rows on
    x = torch.full((1, V), -16.75, dtype=torch.bfloat16)
    x[0, 0] = 0.0
    t = torch.tensor([0])
    res = scoring.token_logprobs(x.repeat(n, 1).to(dev), t.repeat(n).to(dev), 1)
    lp, ent, top_lp, top = OL.token_logprobs(x, t, 1)
    tol, tol_e = OL.tolerances(x, ent)
    off = (res.logprob.cpu().double() - lp).abs().max().item()
    print(f"off by {off * 2 ** 24:.0f} of {tol.item() * 2 ** 24:.0f} half steps")
    assert off <= tol.item() and (res.entropy.cpu().double() - ent).abs().max().item() <= tol_e.item()
    assert (res.top_logprob.cpu().double() - top_lp).abs().max().item() <= tol.item() and bool((res.top_token == 0).all())
