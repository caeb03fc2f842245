"""The 8-bit KV cache: codes and power-of-two scales of key and value vectors, and pages of them.

For the 64 values ``x`` of a token's head: ``e = max(floor(log2 max|x|) - 6, -126)``, ``code = x 2^-e`` rounded to the
nearest (ties to even) and held to [-127, 127], scale byte ``e + 127``; NaN counts as 0, an infinity as the
largest finite bf16.  All in 64 bits, where every step is exact.
"""

from __future__ import annotations

import numpy as np
import torch

LARGEST = float(torch.finfo(torch.bfloat16).max)


def quantise(x: torch.Tensor):
    """``x [..., 64]`` -> (codes int8 ``[..., 64]``, scale bytes uint8 ``[...]``)."""
    x = x.double().nan_to_num(0.0, LARGEST, -LARGEST).numpy()
    top = np.abs(x).max(-1)
    e = np.maximum(np.frexp(top)[1] - 7, -126)  # frexp: top = f 2^k with f in [1/2, 1), so floor(log2 top) = k - 1
    e = np.where(top == 0, -126, e)
    c = np.clip(np.rint(np.ldexp(x, -e[..., None])), -127, 127)
    return torch.from_numpy(c.astype(np.int8)), torch.from_numpy((e + 127).astype(np.uint8))


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """What codes and scale bytes stand for, in 64 bits."""
    return torch.from_numpy(np.ldexp(codes.numpy().astype(np.float64), scales.numpy().astype(np.int64)[..., None] - 127))


def write(pool: torch.Tensor, page: int, slot: int, plane: int, codes: torch.Tensor, scales: torch.Tensor) -> None:
    """One token's codes ``[H, 64]`` and scale bytes ``[H]`` into a slot of ``pool [pages, 2, H, 1040]`` (uint8)."""
    H = pool.shape[2]
    tile = pool[page, plane]
    if plane == 0:
        tile[:, :1024].view(H, 16, 64)[:, slot] = codes.view(torch.uint8)
    else:
        tile[:, :1024].view(H, 64, 16)[:, :, slot] = codes.view(torch.uint8)
    tile[:, 1024 + slot] = scales


def read(pool: torch.Tensor, page: int, slot: int, plane: int) -> torch.Tensor:
    """The values of one slot, ``[H, 64]``."""
    tile, H = pool[page, plane], pool.shape[2]
    codes = tile[:, :1024].contiguous().view(torch.int8)
    codes = codes.view(H, 16, 64)[:, slot] if plane == 0 else codes.view(H, 64, 16)[:, :, slot]
    return values(codes, tile[:, 1024 + slot])
