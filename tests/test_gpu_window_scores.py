"""GPU: windowed attention where every weight is known exactly: large scores beside rising ones, every key of a wide
window counted; and outputs that do not depend on other queries' values."""

import numpy as np
import pytest
import torch

from oracle import window as OW
from yapd_amd import kernels

pytestmark = pytest.mark.gpu
H = 4
LOG2E = np.float32(1.4426950408889634)


def paged(K, V):
    """Dense ``K, V [rows, kv, H, 64]`` (kv a multiple of 16) as a pool and its table."""
    rows, kv = K.shape[:2]
    n = rows * kv // 16
    pool = torch.empty(n, 2, H, 1024, dtype=torch.bfloat16, device=K.device)
    pool[:, 0] = K.reshape(n, 16, H, 64).permute(0, 2, 1, 3).reshape(n, H, 1024)
    pool[:, 1] = V.reshape(n, 16, H, 64).permute(0, 2, 3, 1).reshape(n, H, 1024)
    return pool, torch.arange(n, dtype=torch.int32, device=K.device).view(rows, kv // 16)


def attend(q, K, V, kv, **kw):
    pool, table = paged(K, V)
    out = torch.full_like(q, 77.0)
    kv_len = torch.tensor(kv, dtype=torch.int32, device=q.device)
    kernels.attn_window(q, pool, table, kv_len, out, 0.125, **kw)
    torch.cuda.synchronize()
    return out


def worst_residual(near, scale=0.125):
    """The bf16 value within a factor of two above ``near`` whose product with scale * log2(e) is rounded the most."""
    e = np.float32(2.0 ** np.floor(np.log2(near)))
    a = e * (1 + np.arange(128, dtype=np.float32) / 128)
    c = np.float32(scale) * LOG2E
    off = np.abs(np.float64(a * c) - np.float64(a) * np.float64(c))
    return float(a[off.argmax()])


@pytest.mark.parametrize("parts", [1, 2])
@pytest.mark.parametrize("q_n", [40, 100])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("score", [100, 1000, 2**13, 10**5, 2**20, 2**29])
def test_equal_scores_beside_rising_ones(dev, score, sign, q_n, parts):
    """Query 0's scores are all ``score``; the others' rise by 8 with every 64 keys, so their maxima keep moving.
    V names its keys' 64: query 0 gives 1/64 for each.  In tiles of 128 that is exact: its weights are one bf16 number w,
    their sum 4096 w and each product's 64 w need at most 20 bits, and what remains, 1 / (4096 w) times 64 w, is off by a
    few 2^-24, far below half a step of the result's bf16.  Up to 64 queries the sum is of the weights before their
    rounding to bf16: half a step of theirs, and half a step of the result."""
    kv = 64 * 64
    q = torch.zeros(1, q_n, H, 64)
    q[0, 0, :, 0] = sign * worst_residual(score / 0.125)
    q[0, 1:, :, 1] = 64.0
    K, V = torch.zeros(1, kv, H, 64), torch.zeros(1, kv, H, 64)
    chunk = torch.arange(kv) // 64
    K[..., 0] = 1.0
    K[0, :, :, 1] = chunk[:, None].float()
    V[0, torch.arange(kv), :, chunk] = 1.0
    q, K, V = (x.bfloat16().to(dev) for x in (q, K, V))
    lib = kernels.load_library()
    # the host's bound of the length only decides how the work is cut
    max_kv = 1 if parts == 1 else kv
    assert (lib.yapd_attn_window_workspace(1, q_n, q_n, 0, H, 2 * kv, 0, max_kv) > 0) == (parts > 1)
    out = attend(q, K, V, [kv], window=2 * kv, causal=False, max_kv=max_kv).cpu()
    off = (out[0, 0].double() * 64 - 1).abs().max().item()
    assert off <= (0.0 if q_n > 64 else 2 * 2.0 ** -8 + 1e-4), off
    # the rising ones: half a step of the result's bf16 and of the weights', whose scores of up to 727 are off by 2^-24 of that
    want, a = OW.attend(q[0, 1:2].cpu(), K[0].cpu(), V[0].cpu(), 2 * kv, 0, False, 0.125)
    assert bool(((out[0, 1:].double() - want).abs() <= (2 * 2.0 ** -8 + 1e-4) * a + 1e-6).all())


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("q_n,kv,window", [(30, 320, 100), (64, 640, 1000), (198, 1008, 1000), (198, 1008, 300), (700, 1504, 2000)])
def test_a_query_does_not_depend_on_the_others_values(dev, q_n, kv, window, causal):
    """Half of a row's queries get other values, far larger ones: the bits of the rest stay."""
    g = torch.Generator().manual_seed(q_n)
    K, V = (torch.randn(2, kv, H, 64, generator=g).bfloat16().to(dev) for _ in range(2))
    q = 2 * torch.randn(2, q_n, H, 64, generator=g)
    kw = dict(window=window, sinks=5, causal=causal)
    first = attend(q.bfloat16().to(dev), K, V, [kv, kv - 9], **kw)
    for factor in (0.0, 4.0, 20.0):
        other = q.clone()
        other[:, 1::2] = factor * torch.randn(2, q_n // 2, H, 64, generator=g)
        out = attend(other.bfloat16().to(dev), K, V, [kv, kv - 9], **kw)
        assert torch.equal(out[:, ::2], first[:, ::2])


# (q per row, kv lengths, window, sinks, max_kv): short tiles on four, two and one wave, with parts, tiles of 128 with and without
WIDE = [
    (1, [4000, 1001], 3000, 33, None), (1, [2000] * 250, 1100, 7, None), (1, [1600] * 700, 1500, 0, None),
    (1, [8000], 7000, 64, 8000), (16, [3000, 500], 2500, 4, 1), (33, [2000] * 3, 900, 17, None), (64, [1500] * 20, 1333, 0, None),
    (64, [6000], 5000, 16, 6000), (100, [3000, 777], 2900, 40, 1), (128, [2049, 128], 1999, 100, 1), (300, [6400], 6000, 9, 6400),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("q_n,kv,window,sinks,max_kv", WIDE)
def test_every_key_of_a_wide_window_counts_once(dev, q_n, kv, window, sinks, max_kv, causal):
    """Queries of 0: every visible key weighs the same, exactly 1 before the division.  V names its key's number modulo 64, or its
    64, so an output is a count over N: whole numbers below 2^24, a division off by a few 2^-24 and one rounding to bf16,
    2^-8 of it.  A count is 129 at most here: a key lost or twice there is more."""
    rows, cap = len(kv), (max(kv) + 15) // 16 * 16
    q = torch.zeros(rows, q_n, H, 64, dtype=torch.bfloat16, device=dev)
    j = torch.arange(cap)
    K = torch.randn(1, cap, 1, 64, generator=torch.Generator().manual_seed(0)).bfloat16()
    for name in (j % 64, j // 64 % 64):
        V = torch.nn.functional.one_hot(name, 64).to(torch.bfloat16).view(1, cap, 1, 64)
        Kd, Vd = (x.to(dev).expand(rows, cap, H, 64) for x in (K, V))
        out = attend(q, Kd, Vd, kv, window=window, sinks=sinks, causal=causal, max_kv=max_kv).cpu().double()
        for r in {kv[i]: i for i in range(rows)}.values():  # one of each length
            see = OW.visible(kv[r], q_n, window, sinks, causal).double()
            count = see @ V[0, :kv[r], 0].double()
            assert count.max() <= 129
            want = (count / see.sum(1, keepdim=True))[:, None, :].expand(q_n, H, 64)
            assert bool(((out[r] - want).abs() <= want * (2.0 ** -8 + 1e-6)).all()), (r, name[1].item())
        for r in range(rows):
            assert torch.equal(out[r], out[kv.index(kv[r])])
