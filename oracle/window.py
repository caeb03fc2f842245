"""Attention with a sliding window and sink tokens, one row at a time in 64 bits.

Query ``i`` of a row's last ``n`` positions stands at ``p = kv - n + i`` and sees key ``j`` iff ``j < hi``
and (``j < sinks`` or ``j > p - window``), ``hi = p + 1`` (causal) or ``kv``."""

from __future__ import annotations

import torch


def visible(kv: int, n: int, window: int, sinks: int, causal: bool) -> torch.Tensor:
    """bool ``[n, kv]``: which keys each query sees."""
    p = torch.arange(kv - n, kv)[:, None]
    j = torch.arange(kv)[None, :]
    see = (j < sinks) | (j > p - window)
    return see & (j <= p) if causal else see


def attend(q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, window: int, sinks: int, causal: bool, scale: float):
    """``q [n, H, 64]``, ``K, V [kv, H, 64]`` -> (out ``[n, H, 64]``, ``sum_j w_j |v_j|`` of the same
    shape, which bounds what a relative error of the weights can do).  A query that sees no key: zeros."""
    n, kv = q.shape[0], K.shape[0]
    see = visible(kv, n, window, sinks, causal)
    any_key = see.any(0)
    # a key that no query sees must not matter, whatever it holds
    K = torch.where(any_key[:, None, None], K.double(), 0.0)
    V = torch.where(any_key[:, None, None], V.double(), 0.0)
    s = torch.einsum("qhd,khd->hqk", q.double(), K) * scale
    s = s.masked_fill(~see, -torch.inf)
    m = s.amax(-1, keepdim=True) if kv else s.new_zeros(s.shape[0], n, 1)
    w = torch.exp(s - torch.where(m == -torch.inf, 0.0, m))
    total = w.sum(-1, keepdim=True)
    w = w / torch.where(total > 0, total, 1.0)
    return torch.einsum("hqk,khd->qhd", w, V), torch.einsum("hqk,khd->qhd", w, V.abs())
