"""A windowed attention whose output shares memory with its queries or its pool is refused; one that only lies between or
beside them is not."""

import pytest
import torch

from tests._window_cases import Case
from yapd_amd import kernels

MB = 1 << 20
H, ROW = 4, 4 * 64 * 2  # a token's heads: bytes
Q, POOL, OUT, N_Q = 16 * MB, 64 * MB, 256 * MB, 8
OUT_BYTES, POOL_BYTES = N_Q * ROW, 64 * 2 * H * 1024 * 2

# refused ones only: nothing here may reach a launch, the addresses are nobody's
OVERLAPS = [
    (dict(out=Q), b"overlaps q"), (dict(out=Q + 16), b"overlaps q"), (dict(out=Q - 16), b"overlaps q"),
    (dict(out=Q + (N_Q - 1) * ROW + ROW - 16), b"overlaps q"), (dict(out=Q - OUT_BYTES + 16), b"overlaps q"),
    # queries 20 outputs apart: into the third of them from below and from above, around it
    (dict(stride=20 * OUT_BYTES, out=Q + 40 * OUT_BYTES - OUT_BYTES + 16), b"overlaps q"),
    (dict(stride=20 * OUT_BYTES, out=Q + 40 * OUT_BYTES + ROW - 16), b"overlaps q"),
    (dict(stride=20 * OUT_BYTES, out=Q + 40 * OUT_BYTES - ROW), b"overlaps q"),
    (dict(stride=20 * OUT_BYTES, out=Q + 140 * OUT_BYTES + ROW - 16), b"overlaps q"),
    (dict(out=POOL), b"overlaps the pool"), (dict(out=POOL + POOL_BYTES - 16), b"overlaps the pool"),
    (dict(out=POOL - OUT_BYTES + 16), b"overlaps the pool"), (dict(out=POOL + 1024), b"overlaps the pool"),
]


@pytest.mark.parametrize("change,msg", OVERLAPS)
def test_c_entry_refuses_an_output_that_overlaps(change, msg):
    a = {**dict(q=Q, stride=ROW, out=OUT), **change}
    lib = kernels.load_library()
    rc = lib.yapd_attn_window(a["q"], a["stride"] // 2, POOL, 64, MB, 8, 8, MB, None, 4, 2, N_Q, H, 100, 4, 1, 128, 0.125, None,
                              0, a["out"], None)
    assert rc == 1 and msg in lib.yapd_last_error(), lib.yapd_last_error()


@pytest.mark.gpu
def test_an_output_between_and_beside_queries(dev):
    c = Case(q_lens=[1, 1], kv_lens=[40, 70], H=H, window=30, sinks=3, causal=True)
    t = c.device(dev)
    n = H * 64
    buf = torch.zeros(8 * n, dtype=torch.bfloat16, device=dev)
    q = buf[n:7 * n].view(2, 3 * n)[:, :n].view(2, 1, H, 64)  # tokens n .. 2n and 4n .. 5n

    def run(out):
        q.copy_(t["q"])
        kernels.attn_window(q, t["pool"], t["table"], t["kv_len"], out, 0.125, window=30, sinks=3)
        c.check(out)

    run(buf[2 * n:4 * n].view(2, 1, H, 64))  # exactly between
    run(buf[5 * n:7 * n].view(2, 1, H, 64))  # right behind
    for at in (0, n, 2 * n + 8, 3 * n, 4 * n, 5 * n - 8):
        with pytest.raises(ValueError, match="overlaps q"):
            run(buf[at:at + 2 * n].view(2, 1, H, 64))
    with pytest.raises(ValueError, match="overlaps the pool"):
        run(t["pool"].view(-1)[-2 * n:].view(2, 1, H, 64))
