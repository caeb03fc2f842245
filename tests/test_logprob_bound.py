"""CPU: the bound of the fp32 log probabilities holds for sums in the kernel's order at their worst."""

import numpy as np
import torch

from oracle import logprob as OL


def test_bound_holds_where_a_lane_loses_every_term():
    """One wave a row, 64 lanes of V / 64 terms in sequence: a lane that begins with 1 loses all others, each just below half a step."""
    V, lanes = 34816, 64
    x = torch.full((1, V), -16.75, dtype=torch.float64)
    x[0, 0] = 0.0
    p = np.exp(x[0].numpy()).astype(np.float32).reshape(lanes, V // lanes)
    lane = np.zeros(lanes, dtype=np.float32)
    for i in range(V // lanes):
        lane = lane + p[:, i]
    assert lane[0] == 1.0
    while lane.size > 1:
        lane = lane[: lane.size // 2] + lane[lane.size // 2:]
    lp, ent, _, _ = OL.token_logprobs(x, torch.tensor([0]), 1)
    off = abs(-float(np.log(np.float64(lane[0]))) - lp.item())
    tol = OL.tolerances(x, ent)[0].item()
    assert off > 400 * 2.0 ** -24  # of V / 64 = 544 terms
    assert off <= tol
