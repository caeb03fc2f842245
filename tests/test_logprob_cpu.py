"""CPU: the token-log-probability oracle against torch's log_softmax, and the refusals of the C entry."""

import math

import pytest
import torch

from oracle import logprob as OL
from yapd_amd import kernels


def test_oracle_is_log_softmax():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(6, 50, generator=g, dtype=torch.float64)
    x[1, 3:] = -math.inf
    x[2, 7] = math.nan
    x[3, 9] = math.inf
    t = torch.tensor([4, 1, 0, 0, -1, 50])
    lp, ent, top_lp, top = OL.token_logprobs(x, t, 3)
    want = torch.log_softmax(x, -1)
    assert torch.allclose(lp[:2], want[torch.arange(2), t[:2]]) and bool(lp[2:4].isnan().all())
    assert lp[4] == 0 and bool(lp[5].isnan())
    p = want[[0, 1, 4, 5]].exp()
    assert torch.allclose(ent[[0, 1, 4, 5]], torch.special.entr(p).sum(-1))
    assert torch.equal(top[[0, 4]], x[[0, 4]].topk(3)[1]) and torch.allclose(top_lp[0], want[0].topk(3)[0])
    assert top[1].tolist() == sorted(range(3), key=lambda i: -x[1, i].item())
    assert 7 not in top[2].tolist() and top[3, 0] == 9


def test_oracle_ties_take_the_lowest_index():
    x = torch.zeros(1, 9)
    x[0, ::2] = -0.0
    assert OL.token_logprobs(x, torch.tensor([0]), 4)[3].tolist() == [[0, 1, 2, 3]]


P = 4096
GOOD = dict(logits=P, wide=0, seq=8194, pos=8194, rows=2, bl=3, vocab=8194, tokens=P, k=2, lp=P, ent=P, top_lp=P, top=P,
            stream=None)


@pytest.mark.parametrize("change,msg", [
    (dict(rows=-1), b"rows and bl >= 0"), (dict(rows=2**11, bl=2**11), b"below 2^22"), (dict(vocab=0), b"vocab"),
    (dict(vocab=2**30 + 1), b"vocab"), (dict(k=33), b"top_k"), (dict(k=-1), b"top_k"), (dict(vocab=4, k=5), b"top_k"),
    (dict(logits=None), b"NULL"), (dict(tokens=None), b"NULL"), (dict(top=None), b"NULL"), (dict(lp=None), b"NULL"),
    (dict(logits=P + 1), b"misaligned"), (dict(wide=1, logits=P + 2), b"misaligned"),
])
def test_c_entry_refuses_before_any_launch(change, msg):
    lib = kernels.load_library()
    assert lib.yapd_token_logprobs(*{**GOOD, **change}.values()) == 1
    assert msg in lib.yapd_last_error(), lib.yapd_last_error()


def test_no_positions_launch_nothing():
    assert kernels.load_library().yapd_token_logprobs(*{**GOOD, "rows": 0, "logits": None}.values()) == 0
