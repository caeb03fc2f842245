"""CPU: the windowed attention's oracle against the definition written out, and the refusals of its C entry."""

import pytest
import torch

from oracle import window as OW
from yapd_amd import kernels


@pytest.mark.parametrize("kv,n,window,sinks,causal", [(1, 1, 1, 0, True), (20, 5, 3, 2, True), (20, 5, 3, 2, False),
                                                      (9, 9, 100, 0, True), (12, 4, 1, 50, True), (7, 7, 2, 0, False)])
def test_oracle_is_the_definition(kv, n, window, sinks, causal):
    g = torch.Generator().manual_seed(kv)
    q, K, V = (torch.randn(m, 2, 64, generator=g, dtype=torch.float64) for m in (n, kv, kv))
    out, _ = OW.attend(q, K, V, window, sinks, causal, 0.125)
    for i in range(n):
        p = kv - n + i
        keys = [j for j in range(p + 1 if causal else kv) if j < sinks or j > p - window]
        for h in range(2):
            w = torch.softmax(torch.stack([(q[i, h] * K[j, h]).sum() * 0.125 for j in keys]), 0)
            assert torch.allclose(out[i, h], sum(a * V[j, h] for a, j in zip(w, keys)), atol=1e-12)


def test_oracle_row_without_keys_is_zero():
    out, a = OW.attend(torch.randn(2, 4, 64), torch.empty(0, 4, 64), torch.empty(0, 4, 64), 4, 1, True, 0.125)
    assert bool((out == 0).all()) and bool((a == 0).all())


P = 4096
GOOD = dict(q=P, q_stride=1024, pool=P, n_pages=64, table=P, table_stride=8, table_cols=8, kv_len=P, q_start=None,
            rows=4, max_q=2, n_q=8, n_heads=16, window=100, sinks=4, causal=1, max_kv=128, scale=0.125, ws=None,
            ws_floats=0, out=P, stream=None)


@pytest.mark.parametrize("change,msg", [
    (dict(q=None), b"NULL pointer"), (dict(out=None), b"NULL pointer"), (dict(kv_len=None), b"NULL pointer"),
    (dict(rows=0, n_q=0), b"rows, max_q and n_q >= 1"), (dict(max_q=0), b"rows, max_q and n_q >= 1"),
    (dict(n_heads=6), b"multiple of 4"), (dict(n_heads=0), b"multiple of 4"), (dict(window=0), b"window >= 1"),
    (dict(sinks=-1), b"sinks >= 0"), (dict(max_kv=0), b"max_kv"), (dict(q=P + 8), b"16-byte aligned"),
    (dict(out=P + 2), b"16-byte aligned"), (dict(q_stride=1000), b"q_tok_stride"), (dict(q_stride=1028), b"q_tok_stride"),
    (dict(n_pages=0), b"empty pool"), (dict(table_cols=9), b"empty pool or table"), (dict(n_q=9), b"rows * max_q"),
    (dict(scale=0.0), b"scale"), (dict(scale=-1.0), b"scale"), (dict(scale=float("inf")), b"scale"),
    (dict(scale=1e-31), b"scale"), (dict(scale=1e31), b"scale"), (dict(scale=float("nan")), b"scale"),
    (dict(table_cols=2**27, table_stride=2**27), b"table_cols"),
    (dict(rows=1, max_q=1, n_q=1, n_heads=4, window=20000, max_kv=20000), b"workspace must be"),
    (dict(rows=1, max_q=1, n_q=1, n_heads=4, window=20000, max_kv=20000, ws=P, ws_floats=100), b"workspace must be"),
    (dict(rows=1, max_q=1, n_q=1, n_heads=4, window=20000, max_kv=20000, ws=P + 4, ws_floats=10**9), b"workspace must be"),
    (dict(rows=10**6, max_q=64, n_q=64 * 10**6), b"too many tiles"),
])
def test_c_entry_refuses_before_any_launch(change, msg):
    lib = kernels.load_library()
    assert lib.yapd_attn_window(*{**GOOD, **change}.values()) == 1
    assert msg in lib.yapd_last_error(), lib.yapd_last_error()


def test_workspace_size():
    lib = kernels.load_library()
    assert lib.yapd_attn_window_workspace(256, 1, 256, 0, 16, 1024, 4, 10**6) == 0
    n = lib.yapd_attn_window_workspace(1, 1, 1, 0, 4, 2**30, 2**30, 2**30)
    assert n > 0 and n % (4 * 66) == 0
    assert lib.yapd_attn_window_workspace(1, 1, 1, 0, 5, 100, 0, 100) == -1
