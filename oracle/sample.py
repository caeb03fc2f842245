"""Tokens drawn from logits with given random numbers, one row at a time in 64 bits on the CPU.

Tokens in order (larger logit first, of equal ones the lower index) with weights ``w = exp((x - max) / T)``: the first ``k``,
of those the fewest whose weight is at least ``p`` of theirs, of these the ones of ``w >= m``; the token is the first
whose inclusive sum exceeds ``u`` times the weight kept."""

from __future__ import annotations

import math

import numpy as np
import torch


def sample_row(x: np.ndarray, u: float, T: float, k: int, p: float, m: float):
    """``x [V]`` -> (token, log probability, how near the draw came to another outcome, relative to the weights)."""
    x = np.asarray(x, dtype=np.float64)
    if np.isnan(x).any() or (x == np.inf).any() or (x == -np.inf).all():
        return -1, math.nan, 1.0
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if not T > 0 or k == 1:
        return int(order[0]), 0.0, 1.0
    w = np.exp((x[order] - x[order[0]]) / T)
    margin = 1.0
    if 0 < k < len(w):
        w = w[:int(k)]
    if p < 1:
        c = np.cumsum(w)
        n = int(np.searchsorted(c, max(p, 0.0) * c[-1], side="left"))  # c[n - 1] < p c[-1] <= c[n]
        margin = min(margin, np.abs(c / c[-1] - p).min())
        w = w[:n + 1]
    if m > 0:
        margin = min(margin, np.abs(w - min(m, 1.0)).min())
        w = w[:max(1, int((w >= min(m, 1.0)).sum()))]
    c = np.cumsum(w)
    u = min(max(u if u == u else 0.0, 0.0), 1.0 - 2.0 ** -24)
    n = int(np.searchsorted(c, u * c[-1], side="right"))
    margin = min(margin, np.abs(c / c[-1] - u).min())
    return int(order[n]), math.log(w[n] / c[-1]), margin


def sample_tokens(logits: torch.Tensor, u, T, k, p, m):
    """Rows of ``logits [n, V]`` and settings ``[n]`` -> (token, logprob, margin)."""
    rows = [sample_row(x, *(float(v) for v in s)) for x, s in zip(logits.cpu().double().numpy(), zip(u, T, k, p, m))]
    return (torch.tensor([r[0] for r in rows]), torch.tensor([r[1] for r in rows], dtype=torch.float64),
            torch.tensor([r[2] for r in rows], dtype=torch.float64))


def tolerance(logprob: torch.Tensor) -> torch.Tensor:
    """Bound of |logprob - exact|: the kernel's sums and logarithm are 64-bit (weights off by 2^-38 of the largest at
    most), and one rounding to fp32 follows: 2^-24 of the value; a value near 0 is a difference of two of at most ~100."""
    return logprob.abs() * 2.0 ** -24 + 1e-9
