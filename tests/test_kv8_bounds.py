"""The 8-bit cache's error bounds as they are stated: half a step, which is max|x| / 128 from max|x| = 2^-120 on and 2^-127
for smaller vectors, whose scale is held to 2^-126."""

import pytest
import torch

from oracle import kv8 as OK
from yapd_amd import kernels


def vectors():
    """bf16 vectors of every magnitude, 100 each: the largest value from just above a power of two to just below the next."""
    g = torch.Generator().manual_seed(8)
    out = []
    for k in [*range(-133, -112), -60, 0, 60, *range(120, 128)]:
        x = torch.rand(100, 64, generator=g, dtype=torch.float64) * 2 - 1
        x[:, 0] = torch.linspace(1.0, 255 / 128, 100, dtype=torch.float64)
        out.append((x * 2.0 ** k).to(torch.bfloat16))
    return torch.cat(out)


def check(x, values, scales):
    top = x.double().abs().amax(-1)
    off = (values - x.double()).abs().amax(-1)
    assert bool((off <= torch.pow(2.0, scales.double() - 128)).all())
    large = top >= 2.0 ** -120
    assert bool((off[large] <= top[large] / 128).all())
    assert bool((off[~large] <= 2.0 ** -127).all()) and bool((off[~large] > top[~large] / 128).any())
    assert int(scales.min()) >= 1 and int(scales.max()) <= 248


def test_definition():
    x = vectors()
    codes, scales = OK.quantise(x)
    check(x, OK.values(codes, scales), scales)


@pytest.mark.gpu
def test_kernels(dev):
    x = vectors()
    x = x[:x.shape[0] // 64 * 64].view(-1, 4, 64)
    n = x.shape[0]
    pages = (n + 15) // 16
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    pool8 = torch.zeros(pages, 2, 4, 1040, dtype=torch.uint8, device=dev)
    pool = torch.zeros(pages, 2, 4, 1024, dtype=torch.bfloat16, device=dev)
    table = torch.arange(pages, dtype=torch.int32, device=dev)[None]
    kernels.kv8_write(x.to(dev), x.to(dev), pool8, table, i32([0]))
    kernels.kv8_unpack(pool8, table, i32([n]), pool, table)
    for plane, t in enumerate(kernels.kv_gather(pool, table[0], n)):
        scales = pool8[:, plane, :, 1024:].permute(0, 2, 1).reshape(-1, 4)[:n].cpu()
        check(x.view(-1, 64), t.cpu().double().view(-1, 64), scales.reshape(-1))
