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
    """Bounds of the fp32 pass per row: (for log probabilities, for the entropy), in units of u = 2^-24, half a step.

    Relative to the sum of exponentials, where a row is one wave (at most 4352 granules of 16 bytes, 4 tiles): a lane adds
    V / 64 terms and up to 16 of a granule that the row fills in part; every tile may rescale the sum (an exponential of
    one step = 2 u, and a product: 3 u), the lanes' join once more, with 6 sums; a term has its exponential: V / 64 + 16 +
    12 + 9 + 2.  Where it is eight waves, a lane adds V / 512 + 8 terms in at most V / 18432 + 1 tiles, and the waves'
    join is a rescaling and 8 sums more: V / 512 + 8 + V / 6144 + 3 + 9 + 11 + 2.  Both are below V / 64 + 64.
    Relative to |x - m| (at most 110 where it counts): a term's argument is rounded once, where |m| > 65536 twice, and has
    the constant log2(e), off by 0.3 u; the rescalings' arguments, of |x - m| together, likewise: 5 in all.
    Then x - m, the logarithm (one step), its product with ln 2 and their difference.  The entropy has the logarithm and
    a quotient T / S of at most min(|x - m|, entropy), whose two sums are off by as much each."""
    V = logits.shape[1]
    x = logits.cpu().double()
    m = torch.where(x.isfinite(), x, 0.0).amax(-1)
    far = torch.where(x.isfinite() & (x - m[:, None] > -110), (x - m[:, None]).abs(), 0.0).amax(-1)
    u = 2.0 ** -24
    rel = u * (V / 64 + 64 + 5 * far)
    lp = rel + u * 4 * (far + torch.tensor(float(V)).log() + 1)
    return lp, lp + rel * (far + entropy.nan_to_num(0.0).abs() + 2)
