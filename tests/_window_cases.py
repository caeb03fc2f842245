"""Inputs and tolerances of the windowed-attention tests (plain module, no tests)."""

import numpy as np
import torch

from oracle import window as OW

NAN = float("nan")


def tolerance(o, a):
    """Bound of |kernel - exact| per output.  The weights are rounded to bf16 for the product with V: at most half
    a step, 2^-8 relative, each, so 2^-8 * a with a = sum_j w_j |v_j|; scores, exponentials and sums are fp32
    (64-term products of values up to ~10: relative weight error < 1e-4); the result is rounded to bf16 once: 2^-8 |o|."""
    half = torch.finfo(torch.bfloat16).eps / 2
    e = (half + 1e-4) * a
    return e + half * (o.abs() + e) + 1e-30


class Case:
    """Rows of a paged cache whose pages and slots that no query sees hold NaN, and whose table
    entries of pages that no query sees are out of range."""

    def __init__(self, *, q_lens, kv_lens, H, window, sinks, causal, seed=0, packed=False, tail_q=0, extra_cols=1):
        g = torch.Generator().manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.q_lens, self.kv_lens, self.H = list(q_lens), list(kv_lens), H
        self.window, self.sinks, self.causal, self.packed = window, sinks, causal, packed
        rows = len(q_lens)
        cols = max(1, max((x + 15) // 16 for x in kv_lens)) + extra_cols
        n_pages = sum((x + 15) // 16 for x in kv_lens) + 3
        order = rng.permutation(n_pages)
        table = rng.choice([-5, n_pages, 2**31 - 1, -2**31], size=(rows, cols)).astype(np.int64)
        pool = torch.full((n_pages, 2, H, 1024), NAN, dtype=torch.bfloat16)
        self.n_q = sum(q_lens) + tail_q
        self.q = (2 * torch.randn(self.n_q, H, 64, generator=g)).bfloat16()
        self.starts = [int(x) for x in np.concatenate([[0], np.cumsum(q_lens)])]
        self.ref = torch.zeros(self.n_q, H, 64, dtype=torch.float64)
        self.tol = torch.zeros(self.n_q, H, 64, dtype=torch.float64)
        at = 0
        for r, (n, kv) in enumerate(zip(q_lens, kv_lens)):
            if kv == 0:
                continue
            npg = (kv + 15) // 16
            K = torch.randn(npg * 16, H, 64, generator=g).bfloat16()
            V = torch.randn(npg * 16, H, 64, generator=g).bfloat16()
            see = OW.visible(kv, n, window, sinks, causal).any(0) if n else torch.zeros(kv, dtype=torch.bool)
            see = torch.cat([see, torch.zeros(npg * 16 - kv, dtype=torch.bool)])
            K[~see] = NAN
            V[~see] = NAN
            pages = order[at:at + npg]
            at += npg
            used = see.view(npg, 16).any(1)
            table[r, :npg][used.numpy()] = pages[used.numpy()]
            pg = torch.from_numpy(pages)
            pool[pg, 0] = K.view(npg, 16, H, 64).permute(0, 2, 1, 3).reshape(npg, H, 1024)
            pool[pg, 1] = V.view(npg, 16, H, 64).permute(0, 2, 3, 1).reshape(npg, H, 1024)
            if n:
                s = slice(self.starts[r], self.starts[r + 1])
                o, a = OW.attend(self.q[s], K[:kv], V[:kv], window, sinks, causal, 0.125)
                self.ref[s], self.tol[s] = o, tolerance(o, a)
        self.pool, self.table = pool, torch.from_numpy(table.astype(np.int32))

    def device(self, dev):
        d = lambda x: x.to(dev)  # noqa: E731
        q = self.q if self.packed else self.q.view(len(self.q_lens), self.q_lens[0], self.H, 64)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
        return dict(q=d(q), pool=d(self.pool), table=d(self.table), kv_len=i32(self.kv_lens),
                    q_start=i32(self.starts) if self.packed else None)

    def run(self, dev, kernels, **kw):
        t = self.device(dev)
        out = torch.full_like(t["q"], 77.0)
        kernels.attn_window(t["q"], t["pool"], t["table"], t["kv_len"], out, 0.125, window=self.window,
                            sinks=self.sinks, causal=self.causal, q_start=t["q_start"], **kw)
        torch.cuda.synchronize()
        return out

    def check(self, out):
        out = out.cpu().double().view(self.n_q, self.H, 64)
        n = self.starts[-1]
        assert bool((out[n:] == 77.0).all()), "rows behind the last sequence were written"
        err = (out[:n] - self.ref[:n]).abs()
        bad = ~(err <= self.tol[:n])  # NaN fails too
        assert not bool(bad.any()), (f"{int(bad.sum())} of {bad.numel()} values off, first at {bad.nonzero()[0].tolist()}, "
                                     f"worst {err.nan_to_num(1e9).max().item():.4g}")
