"""The cache of shared pages, the attention that reads it and the log probabilities that rank what was
decoded from it, used together: prompts, candidates forked from them, steps behind a window, a winner."""

import pytest
import torch

from oracle import logprob as OL
from oracle import window as OW
from tests._window_cases import tolerance
from yapd_amd import kernels
from yapd_amd.paged import SharedPagedKV
from yapd_amd.scoring import token_logprobs

pytestmark = pytest.mark.gpu

H, LAYERS, VOCAB = 4, 2, 203
WINDOW, SINKS = 48, 5
SCALE = 0.125


class Decoder:
    """Rows with random Q, K, V per position and layer: what they hold is kept densely on the CPU too."""

    def __init__(self, dev, n_rows, n_pages):
        self.dev, self.gen = dev, torch.Generator().manual_seed(3)
        self.kv = SharedPagedKV(n_layers=LAYERS, n_rows=n_rows, pages_per_row=20, n_heads=H, device=dev, n_pages=n_pages)
        for pool in self.kv.pools:
            pool.fill_(float("nan"))  # what was never written is never used
        self.k = [[torch.empty(0, H, 64) for _ in range(LAYERS)] for _ in range(n_rows)]
        self.v = [[torch.empty(0, H, 64) for _ in range(LAYERS)] for _ in range(n_rows)]

    def length(self, row):
        return self.k[row][0].shape[0]

    def draw(self, *shape):
        return torch.randn(*shape, generator=self.gen).bfloat16()

    def append(self, rows, n):
        """``n[i]`` new positions of ``rows[i]`` in every layer, written one row at a time."""
        for row, count in zip(rows, n):
            at = self.length(row)
            self.kv.reserve(row, at, at + count)
            pos0 = torch.tensor([at], dtype=torch.int32, device=self.dev)
            for layer, pool in enumerate(self.kv.pools):
                k, v = self.draw(count, H, 64), self.draw(count, H, 64)
                self.k[row][layer] = torch.cat([self.k[row][layer], k])
                self.v[row][layer] = torch.cat([self.v[row][layer], v])
                kernels.kv_write(k.to(self.dev), v.to(self.dev), pool, self.kv.table[row:row + 1], pos0, count)

    def fork(self, src, dst):
        self.kv.fork(src, dst, self.length(src))
        for r in dst:
            self.k[r], self.v[r] = list(self.k[src]), list(self.v[src])

    def attend(self, rows, n, packed, causal=True):
        """The last ``n[i]`` positions of ``rows[i]``, checked in every layer; returns the last layer's output."""
        q = self.draw(sum(n), H, 64)
        table = self.kv.table[torch.tensor(rows, device=self.dev)].contiguous()
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=self.dev)  # noqa: E731
        kv_len = i32([self.length(r) for r in rows])
        starts = [sum(n[:i]) for i in range(len(n) + 1)]
        qd = q.to(self.dev) if packed else q.to(self.dev).view(len(rows), n[0], H, 64)
        for layer, pool in enumerate(self.kv.pools):
            out = torch.empty_like(qd)
            kernels.attn_window(qd, pool, table, kv_len, out, SCALE, window=WINDOW, sinks=SINKS, causal=causal,
                                q_start=i32(starts) if packed else None)
            got = out.cpu().double().view(-1, H, 64)
            for i, row in enumerate(rows):
                s = slice(starts[i], starts[i + 1])
                want, a = OW.attend(q[s], self.k[row][layer], self.v[row][layer], WINDOW, SINKS, causal, SCALE)
                assert bool(((got[s] - want).abs() <= tolerance(want, a)).all()), (row, layer)
        return out.view(-1, H * 64)

    def behind(self, row):
        """Give back what the next query's window no longer sees."""
        self.kv.release_before(row, self.length(row) + 1 - WINDOW, SINKS)


def score(hidden, head, tokens):
    logits = (hidden.float() @ head).bfloat16()
    res = token_logprobs(logits, tokens, top_k=4)
    lp, entropy, top_lp, top = OL.token_logprobs(logits, tokens, 4)
    t_lp, t_ent = OL.tolerances(logits, entropy)
    assert bool(((res.logprob.cpu().double() - lp).abs() <= t_lp).all())
    assert bool(((res.entropy.cpu().double() - entropy).abs() <= t_ent).all())
    assert bool(((res.top_logprob.cpu().double() - top_lp).abs() <= t_lp[:, None]).all())
    assert bool((res.top_token.cpu() == top).all())
    return res


def test_prompts_candidates_and_a_winner(dev):
    d = Decoder(dev, n_rows=6, n_pages=90)
    head = torch.randn(H * 64, VOCAB, generator=d.gen).to(dev)
    # three prompts at once, packed
    d.append([0, 1, 2], [70, 33, 130])
    d.attend([0, 1, 2], [70, 33, 130], packed=True)
    assert d.kv.free_pages == 89 - 5 - 3 - 9
    # row 1 gives three candidates: two whole pages shared, the third copied
    d.fork(1, [3, 4, 5])
    assert d.kv.free_pages == 89 - 17 - 3
    rows, total = [1, 3, 4, 5], torch.zeros(4, dtype=torch.float64)
    for step in range(70):  # past the window: pages are given back on the way
        d.append(rows, [1] * 4)
        hidden = d.attend(rows, [1] * 4, packed=False)
        tokens = torch.randint(0, VOCAB, (4,), generator=d.gen).to(dev)
        total += score(hidden, head, tokens).logprob.cpu().double()
        for r in rows:
            d.behind(r)
    # of 103 positions 6 pages at most: the sinks' and the window's
    assert all((d.kv.table_host[r] != 0).sum() <= 5 for r in rows)
    best = rows[int(total.argmax())]
    for r in rows:
        if r != best:
            d.kv.release(r)
            d.k[r], d.v[r] = [torch.empty(0, H, 64)] * LAYERS, [torch.empty(0, H, 64)] * LAYERS
    d.kv.release(0)
    # the winner and the untouched row 2 move to the front and go on as before, the winner with a block
    used = d.kv.compact()
    assert used == 1 + 9 + (d.kv.table_host[best] != 0).sum() and d.kv.table_host.max() == used - 1
    d.append([best, 2], [20, 20])
    hidden = d.attend([best, 2], [20, 20], packed=False, causal=False)
    score(hidden, head, torch.randint(-1, VOCAB, (40,), generator=d.gen).to(dev))


def test_captured_step_follows_a_cache_that_changes(dev):
    """One captured attention step over a cache whose rows grow, fork, lose pages and are compacted."""
    d = Decoder(dev, n_rows=4, n_pages=60)
    d.append([0, 1], [60, 18])
    q = torch.zeros(4, 1, H, 64, dtype=torch.bfloat16, device=dev)
    out = torch.empty_like(q)
    kv_len = torch.zeros(4, dtype=torch.int32, device=dev)

    def step():
        kernels.attn_window(q, d.kv.pools[1], d.kv.table, kv_len, out, SCALE, window=WINDOW, sinks=SINKS)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for turn in range(6):
        if turn == 1:
            d.fork(0, [2])
        if turn == 3:
            d.kv.release(1)
            d.k[1], d.v[1] = [torch.empty(0, H, 64)] * LAYERS, [torch.empty(0, H, 64)] * LAYERS
        if turn == 4:
            d.kv.compact()
        rows = [r for r in range(4) if d.length(r)]
        d.append(rows, [7] * len(rows))
        for r in rows:
            d.kv.release_before(r, d.length(r) - WINDOW, SINKS)
        new_q = d.draw(4, 1, H, 64)
        q.copy_(new_q)
        kv_len.copy_(torch.tensor([d.length(r) for r in range(4)], dtype=torch.int32))
        out.fill_(77.0)
        g.replay()
        torch.cuda.synchronize()
        for r in range(4):
            want, a = OW.attend(new_q[r], d.k[r][1], d.v[r][1], WINDOW, SINKS, True, SCALE)
            assert bool(((out[r].cpu().double() - want).abs() <= tolerance(want, a)).all()), (turn, r)
