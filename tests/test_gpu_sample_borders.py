"""GPU: draws whose target lies between two sums of the same elements, added up in different orders.

The inputs were searched for: with 512 threads a row, a prefix sum that adds its lanes up in an order of their own makes the
sums before and behind a thread without elements differ by one rounding, and these targets lie in between.  Either side of
the border is right; a token that is no token of the row is not."""

import math

import numpy as np
import pytest
import torch

from yapd_amd import kernels

pytestmark = pytest.mark.gpu

V = 60
# (seed of the row, temperature, number): the number is u, or top-p with the last kept token drawn
UNIFORM = [(68, 0.640668511390686, 0.4193077087402344), (152, 0.927489161491394, 0.8685406446456909),
           (192, 1.7711901664733887, 0.5916163921356201), (232, 1.9186112880706787, 0.5243672132492065),
           (248, 0.658687949180603, 0.9049968719482422), (524, 1.0126303434371948, 0.3403594493865967),
           (552, 1.1445252895355225, 0.7578786015510559), (564, 1.7868139743804932, 0.5833597779273987),
           (616, 1.2523404359817505, 0.3996359407901764), (776, 0.6378098726272583, 0.7938340306282043),
           (836, 0.8197837471961975, 0.9949377775192261), (888, 1.2790608406066895, 0.9815874695777893)]
TOP_P = [(192, 1.8448772430419922, 0.5836614966392517), (652, 1.558657169342041, 0.5861777067184448),
         (720, 0.5884726047515869, 0.8869616985321045), (756, 0.9813641309738159, 0.9975509643554688),
         (832, 0.8591547608375549, 0.8144136071205139)]


@pytest.mark.parametrize("by_top_p", [False, True])
def test_targets_between_two_sums_of_the_same_elements(dev, by_top_p):
    cases = TOP_P if by_top_p else UNIFORM
    n = len(cases)
    rows = [torch.randn(V, generator=torch.Generator().manual_seed(s)).bfloat16() for s, _, _ in cases]
    x = torch.zeros(n, 64, dtype=torch.bfloat16, device=dev)[:, :V]
    x.copy_(torch.stack(rows))
    T = torch.tensor([t for _, t, _ in cases], device=dev)
    number = torch.tensor([v for _, _, v in cases], device=dev)
    one = torch.ones(n, device=dev)
    token = torch.full((n,), -7, dtype=torch.int64, device=dev)
    logprob = torch.full((n,), 55.0, device=dev)
    kernels.sample_tokens(x, one if by_top_p else number, token, logprob, temperature=T, top_p=number if by_top_p else 1.0)
    for i, (_, t, v) in enumerate(cases):
        values = rows[i].double().numpy()
        order = np.argsort(-values, kind="stable")
        w = np.exp((values[order] - values[order[0]]) / float(T[i]))
        c = np.cumsum(w)
        at = int(np.abs(c / c[-1] - v).argmin())  # v is the share of the first at + 1 elements
        assert abs(c[at] / c[-1] - v) < 1e-14
        got = int(token[i])
        assert got in (order[at], order[at + 1]), (i, got)
        j = int(np.nonzero(order == got)[0][0])
        want = math.log(w[j] / (c[j] if by_top_p else c[-1]))
        assert abs(float(logprob[i]) - want) <= abs(want) * 2.0 ** -24 + 1e-9
