"""Log probabilities of given tokens, entropy and best alternatives in 64 bits."""

from __future__ import annotations

import torch


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, k: int):
    """``logits [n, V]``, ``tokens [n]`` -> (logprob, entropy, top logprob ``[n, k]``, top token ``[n, k]``) on
    the CPU.  A token below 0: 0; one past the vocabulary: NaN.  Top: value, then lowest index; NaN as -inf."""
    x = logits.cpu().double()
    tokens = tokens.cpu()
    V = x.shape[1]
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    log_s = e.sum(-1).log()
    d = torch.where(e == 0, 0.0, x - m)  # p = 0 adds nothing; NaN stays
    entropy = log_s - (d * e).sum(-1) / e.sum(-1)
    lp_all = (x - m) - log_s[:, None]
    lp = lp_all.gather(1, tokens.clamp(0, V - 1)[:, None])[:, 0]
    lp = torch.where(tokens < 0, 0.0, torch.where(tokens >= V, torch.nan, lp))
    order = torch.where(x.isnan(), -torch.inf, x + 0.0)
    top = torch.sort(order, dim=-1, descending=True, stable=True)[1][:, :k]
    return lp, entropy, lp_all.gather(1, top), top


def tolerances(logits: torch.Tensor, entropy: torch.Tensor):
    """Bounds of the fp32 pass per row: (for log probabilities, for the entropy).  In units of 2^-24, half a step:
    a lane adds V / 256 terms and about 64 joins follow, each term with an exponential of one step, an argument
    rounded twice (|x - m| <= 104 where it counts) -- relative to the sum of exponentials; then x - m, the
    logarithm and their difference, each rounded once."""
    V = logits.shape[1]
    x = logits.cpu().double()
    m = torch.where(x.isfinite(), x, 0.0).amax(-1)
    far = torch.where(x.isfinite() & (x - m[:, None] > -110), (x - m[:, None]).abs(), 0.0).amax(-1)
    u = 2.0 ** -24
    rel = u * (V / 256 + 64 + 3 * far)
    lp = rel + u * 4 * (far + torch.tensor(float(V)).log() + 1)
    return lp, lp + rel * (far + entropy.nan_to_num(0.0).abs() + 2)
