"""Attention for a tree of drafted tokens over a row's keys, one row at a time in 64 bits.

The row's last ``n`` keys are its nodes, ``ctx = kv - n``.  Node ``i`` sees node ``j`` iff bit ``j`` of its mask is set, and
key ``j < ctx`` iff ``j < sinks`` or ``j > ctx + depth - window``, ``depth`` the other bits set in its mask."""

from __future__ import annotations

from typing import Optional, Sequence

import torch


def visible(kv: int, n: int, masks: Sequence[int], window: Optional[int], sinks: int) -> torch.Tensor:
    """bool ``[len(masks), kv]``: which keys each of a row's first nodes sees."""
    ctx = kv - n
    see = torch.zeros(len(masks), kv, dtype=torch.bool)
    for i, bits in enumerate(masks):
        bits = int(bits) & (2 ** min(n, 64) - 1)
        depth = bin(bits & ~(1 << i)).count("1")
        for j in range(kv):
            if j < ctx:
                see[i, j] = window is None or j < sinks or j > ctx + depth - window
            else:
                see[i, j] = bool(bits >> (j - ctx) & 1)
    return see


def attend(q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, see: torch.Tensor, scale: float):
    """``q [n, H, 64]``, ``K, V [kv, H, 64]``, ``see [n, kv]`` -> (out, sum of weights times |V|), both ``[n, H, 64]``; zeros where
    nothing is seen.  What a node does not see never enters, whatever it holds."""
    out = torch.zeros(q.shape, dtype=torch.float64)
    mag = torch.zeros_like(out)
    for i in range(q.shape[0]):
        k, v = K[see[i]].double(), V[see[i]].double()
        if not len(k):
            continue
        w = torch.softmax(torch.einsum("hd,khd->hk", q[i].double(), k) * scale, -1)
        out[i] = torch.einsum("hk,khd->hd", w, v)
        mag[i] = torch.einsum("hk,khd->hd", w, v.abs())
    return out, mag
