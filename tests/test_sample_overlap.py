"""yapd_sample_tokens refuses outputs that share memory with an input, before any GPU call: rows are drawn side by side,
and a row's output written into another row's logits or settings would change that row's draw."""

import pytest
import torch

from yapd_amd import kernels, scoring

V, ROWS, BL, PITCH = 50, 3, 4, 64  # bf16: rows of 100 bytes, 128 apart, 12 of them
N = ROWS * BL
X, U, T, K, P, M, TOKEN, LP = (0x10000 * i for i in range(1, 9))
CALL = dict(logits=X, wide=0, seq=BL * PITCH, pos=PITCH, rows=ROWS, bl=BL, vocab=V, u=U, t=T, t_all=1.0, k=K, k_all=0, p=P,
            p_all=1.0, m=M, m_all=0.0, token=TOKEN, logprob=LP, stream=None)


@pytest.mark.parametrize("over,msg", [
    (dict(logprob=U), b"settings"), (dict(logprob=T), b"settings"), (dict(logprob=K), b"settings"), (dict(logprob=P), b"settings"),
    (dict(logprob=M + 4 * (N - 1)), b"settings"), (dict(token=U - 8 * N + 4), b"settings"), (dict(token=T + 4), b"settings"),
    (dict(token=LP + 4 * (N - 1)), b"overlap"), (dict(token=LP - 8 * N + 4), b"overlap"),
    (dict(logprob=X), b"logits"), (dict(token=X + (N - 1) * 128 + 96), b"logits"), (dict(logprob=X - 4 * N + 2), b"logits"),
    (dict(seq=-BL * PITCH, logprob=X - 2 * BL * 128 + 96), b"logits"),       # rows that go down in memory
    (dict(seq=0, pos=0, logprob=X + 96), b"logits"),                         # one row for all
    (dict(wide=1, logprob=X + (N - 1) * 256 + 196), b"logits"),
    (dict(rows=1, bl=1, token=X + 96), b"logits"),
])
def test_refuses(over, msg):
    lib = kernels.load_library()
    assert lib.yapd_sample_tokens(*dict(CALL, **over).values()) == 1
    assert msg in lib.yapd_last_error()


@pytest.mark.gpu
def test_outputs_between_the_rows(dev):
    """Outputs in the bytes behind rows of a padded pitch share none with a row."""
    buf = torch.zeros(3, PITCH, dtype=torch.bfloat16, device=dev)
    x = buf[:, :V]
    x.copy_(torch.randn(3, V, generator=torch.Generator().manual_seed(0)))
    token = buf.view(-1)[52:64].view(torch.int64)   # bytes 104 to 127 of row 0's 128
    logprob = buf.view(-1)[PITCH + 50:PITCH + 56].view(torch.float32)
    u = torch.tensor([0.1, 0.5, 0.9], device=dev)
    want = scoring.sample_tokens(x, u)
    kernels.sample_tokens(x, u, token, logprob)
    assert torch.equal(token, want.token) and torch.equal(logprob, want.logprob)
    with pytest.raises(ValueError, match="settings"):
        kernels.sample_tokens(x, u, want.token, u)
    with pytest.raises(ValueError, match="logits"):
        kernels.sample_tokens(x, u, buf.view(-1)[48:60].view(torch.int64), want.logprob)
