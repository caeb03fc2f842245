"""The operators of long-form generation with candidates, as timed cases: attention with a sliding
window and sink tokens over the paged KV cache, copies of cache pages in every layer, and log
probabilities of given tokens with entropy and the best alternatives.

Where ``own`` is false, ``run`` computes an operator from elementary torch operations in 32 bits; where
it is true, it makes the call a user of the package makes.  ``exact`` is the same result in 64 bits.

Shapes are the T3 backbone's (16 heads of 64, 30 layers, 16-token pages, speech vocabulary 8194) with
generic ones beside them.  Sequence lengths are the mid-quantiles of their distribution, shuffled by the
seed: every seed has other rows but the same total, so ``work`` is exact without the seed.
"""

from __future__ import annotations

import math
import random
from types import SimpleNamespace

import numpy as np
import torch

own = False

PAGE, HD = 16, 64
SCALE = 0.125
BF = torch.bfloat16


def listed():
    return [
        # One stream's next token behind a window: the smallest call, latency counts.
        dict(name="token_one", op="window", rows=1, q_lo=1, q_hi=1, past_lo=1500, past_hi=1500, window=1024, sinks=4,
             causal=True, heads=16),
        # A server's single-token step: many streams, very uneven lengths, most of them past the window.
        dict(name="token_batch", op="window", rows=256, q_lo=1, q_hi=1, past_lo=60, past_hi=4000, window=1024, sinks=64,
             causal=True, heads=16),
        # A block-diffusion step of long utterances: blocks of 32, bidirectional, odd window and sinks.
        dict(name="block_ragged", op="window", rows=130, q_lo=32, q_hi=32, past_lo=100, past_hi=2000, window=500,
             sinks=33, causal=False, heads=16),
        # A few streams with a window of most of a long cache: too few rows to fill the chip.
        dict(name="token_long", op="window", rows=3, q_lo=1, q_hi=1, past_lo=20000, past_hi=30000, window=16384,
             sinks=16, causal=True, heads=16),
        # Prompts of several requests prefilled at once, packed back to back, each in an empty row.
        dict(name="prompts_packed", op="window", rows=9, q_lo=70, q_hi=1500, past_lo=0, past_hi=0, window=512, sinks=16,
             causal=True, heads=16),
        # One long text: 8000 tokens on top of an earlier part.
        dict(name="prompt_long", op="window", rows=1, q_lo=8000, q_hi=8000, past_lo=1000, past_hi=1000, window=2048,
             sinks=64, causal=True, heads=16),
        # A fork: the partial last page of one row, in every layer.
        dict(name="copy_fork", op="copy", pairs=1, pages=64, layers=30, heads=16, shared=False),
        # A prefix of 19 pages copied to seven candidates' rows (sources repeat).
        dict(name="copy_prefix", op="copy", pairs=133, pages=256, layers=30, heads=16, shared=True),
        # Compaction of a pool: every live page behind the gap moves into a hole.
        dict(name="copy_compact", op="copy", pairs=301, pages=640, layers=30, heads=16, shared=False),
        # A block's 32 positions of one pair, tokens just decided.
        dict(name="logprob_block", op="logprob", rows=64, vocab=8194, top=8, wide=False, masked=False),
        # Every position of the 256-pair step, some vocabulary entries masked out.
        dict(name="logprob_step", op="logprob", rows=16384, vocab=8194, top=4, wide=False, masked=True),
        # A large vocabulary of odd size in fp32.
        dict(name="logprob_wide", op="logprob", rows=900, vocab=100003, top=20, wide=True, masked=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["token", "token", "block", "prompt", "copy", "logprob", "logprob"])
    if op == "token":
        rows, window = _log_int(rng, 1, 300), _log_int(rng, 33, 8000)
        window = min(window, 200000 // rows)
        lo = _log_int(rng, 1, 3000)
        return dict(op="window", rows=rows, q_lo=1, q_hi=1, past_lo=lo, past_hi=min(lo * rng.randint(1, 8), 12000),
                    window=window, sinks=rng.choice([0, 1, 4, 16, 31, 64]), causal=True, heads=rng.choice([4, 8, 16, 16]))
    if op == "block":
        rows, bl = _log_int(rng, 1, 150), rng.choice([5, 8, 16, 16, 32, 32, 48, 64])
        lo = _log_int(rng, 10, 1000)
        return dict(op="window", rows=rows, q_lo=bl, q_hi=bl, past_lo=lo, past_hi=lo * rng.randint(1, 4),
                    window=_log_int(rng, 17, 1500), sinks=rng.choice([0, 3, 16, 33, 100]),
                    causal=rng.choice([False, False, True]), heads=rng.choice([4, 8, 16, 16]))
    if op == "prompt":
        rows = _log_int(rng, 1, 12)
        hi = _log_int(rng, 100, 8000 // rows)
        past = rng.choice([0, 0, rng.randint(1, 1500)])
        return dict(op="window", rows=rows, q_lo=rng.randint(1, hi), q_hi=hi, past_lo=past, past_hi=past,
                    window=_log_int(rng, 33, 2000), sinks=rng.choice([0, 4, 17, 64]),
                    causal=hi > 1000 or rng.choice([True, False]), heads=rng.choice([4, 8, 16, 16]))
    if op == "copy":
        pairs = _log_int(rng, 1, 250)
        return dict(op="copy", pairs=pairs, pages=2 * pairs + rng.randint(1, 100), layers=rng.choice([1, 12, 30, 30]),
                    heads=rng.choice([4, 8, 16, 16]), shared=rng.choice([False, True]))
    wide = rng.choice([False, False, True])
    vocab = rng.choice([8194, 8194, _log_int(rng, 100, 100000)])
    rows = _log_int(rng, 1, min(16384, (80 if wide else 130) * 1000 * 1000 // vocab))
    return dict(op="logprob", rows=rows, vocab=vocab, top=rng.choice([1, 1, 4, 5, 10, 20, 32]), wide=wide,
                masked=rng.choice([False, True]))


# --------------------------------------------------------------------------- inputs

def _lengths(n, lo, hi, seed=None):
    """n lengths in [lo, hi] at the mid-quantiles of a uniform distribution, shuffled by the seed."""
    out = [int(round(lo + (hi - lo) * (i + 0.5) / n)) for i in range(n)]
    if seed is not None:
        random.Random(seed).shuffle(out)
    return out


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape, std=1.0, dtype=BF):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def prepare(case, seed):
    return {"window": _prepare_window, "copy": _prepare_copy, "logprob": _prepare_logprob}[case["op"]](case, seed)


def _prepare_window(case, seed):
    g, H, rows = _gen(seed), case["heads"], case["rows"]
    q_len = _lengths(rows, case["q_lo"], case["q_hi"], seed)
    past = _lengths(rows, case["past_lo"], case["past_hi"], seed + 1)
    kv_len = [a + b for a, b in zip(past, q_len)]
    cols = (max(kv_len) + PAGE - 1) // PAGE
    n_pages = sum((x + PAGE - 1) // PAGE for x in kv_len) + 8
    order = np.random.default_rng(seed).permutation(n_pages).astype(np.int32)
    table, at = np.zeros((rows, cols), dtype=np.int32), 0
    for r, x in enumerate(kv_len):
        n = (x + PAGE - 1) // PAGE
        table[r, :n] = order[at:at + n]
        at += n
    pool = torch.empty(n_pages, 2, H, PAGE * HD, dtype=BF, device="cuda").normal_(generator=g)
    packed = case["q_lo"] != case["q_hi"] or case["q_hi"] > 64
    n_q = sum(q_len)
    q_start = [0]
    for x in q_len:
        q_start.append(q_start[-1] + x)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    # queries with some spread, so that a softmax has weight on a few keys
    q = _normal(g, n_q, H, HD, std=2.0)
    return SimpleNamespace(op="window", q=q if packed else q.view(rows, case["q_hi"], H, HD), pool=pool,
                           table=torch.from_numpy(table).cuda(), kv_len=ints(kv_len), q_start=ints(q_start),
                           packed=packed, max_q=max(q_len), max_kv=max(kv_len), window=case["window"],
                           sinks=case["sinks"], causal=case["causal"], kv_host=kv_len, q_host=q_len)


def _prepare_copy(case, seed):
    g = _gen(seed)
    pools = [torch.empty(case["pages"], 2, case["heads"], PAGE * HD, dtype=BF, device="cuda").normal_(generator=g)
             for _ in range(case["layers"])]
    order = np.random.default_rng(seed).permutation(case["pages"]).astype(np.int32)
    n = case["pairs"]
    src = np.resize(order[n:n + _sources(case)], n)
    return SimpleNamespace(op="copy", pools=pools, src=src, dst=order[:n].copy())


def _sources(case):
    return (case["pairs"] + 6) // 7 if case["shared"] else case["pairs"]


def _prepare_logprob(case, seed):
    g, rows, V = _gen(seed), case["rows"], case["vocab"]
    pitch = (V + 7) // 8 * 8  # rows as the speech head leaves them: padded to 16 bytes
    x = torch.empty(rows, pitch, dtype=torch.float32 if case["wide"] else BF, device="cuda")
    x.normal_(std=3.0, generator=g)
    logits = x[:, :V]
    tokens = torch.randint(0, V, (rows,), generator=g, device="cuda")
    if case["masked"]:
        # an eighth of the vocabulary is not allowed; a token that was drawn is
        off = torch.rand(V, generator=g, device="cuda") < 0.125
        keep = logits.gather(1, tokens[:, None])
        logits[:, off] = -math.inf
        logits.scatter_(1, tokens[:, None], keep)
    return SimpleNamespace(op="logprob", logits=logits, tokens=tokens, top=case["top"])


# --------------------------------------------------------------------------- one pass

def run(state):
    if own:
        return {"window": _own_window, "copy": _own_copy, "logprob": _own_logprob}[state.op](state)
    return {"window": _plain_window, "copy": _plain_copy, "logprob": _plain_logprob}[state.op](state)


def _own_window(s):
    from yapd_amd import kernels
    out = torch.empty_like(s.q)
    kernels.attn_window(s.q, s.pool, s.table, s.kv_len, out, SCALE, window=s.window, sinks=s.sinks, causal=s.causal,
                        q_start=s.q_start if s.packed else None, max_q=s.max_q, max_kv=s.max_kv)
    return out


def _own_copy(s):
    from yapd_amd import kernels
    kernels.kv_copy_pages(s.pools, s.src, s.dst)
    return s.pools


def _own_logprob(s):
    from yapd_amd import scoring
    r = scoring.token_logprobs(s.logits, s.tokens, top_k=s.top)
    return r.logprob, r.entropy, r.top_logprob, r.top_token


def _plain_window(s):
    """The keys a row's queries can see, gathered from the pages (the sinks, then everything from the
    first query's window on), one masked softmax over them, in 32 bits."""
    H, dev = s.pool.shape[2], s.pool.device
    rows, Q = s.kv_len.numel(), s.max_q
    kv, start = s.kv_len.long(), s.q_start.long()
    qn = start[1:] - start[:-1]
    i = torch.arange(Q, device=dev)
    live = i[None, :] < qn[:, None]                                   # [rows, Q]
    at = (start[:-1, None] + i).clamp_max(s.q.numel() // (H * HD) - 1)
    q = s.q.reshape(-1, H, HD)[at].float()                            # [rows, Q, H, 64]
    p = (kv - qn)[:, None] + i                                        # the queries' positions
    first = (kv - qn - s.window + 1).clamp_min(s.sinks)               # first key behind the sinks
    span = min(s.max_kv, s.window + Q)
    sink = torch.arange(s.sinks, device=dev).expand(rows, -1)
    j = torch.cat([sink, first[:, None] + torch.arange(span, device=dev)], 1)  # [rows, N] key positions
    there = j < kv[:, None]
    jc = torch.where(there, j, 0)
    page = torch.gather(s.table.long(), 1, jc // PAGE)
    slot = jc % PAGE
    kp = s.pool[:, 0].view(-1, H, PAGE, HD)
    vp = s.pool[:, 1].view(-1, H, HD, PAGE)
    k = kp[page, :, slot].float()                                     # [rows, N, H, 64]
    v = vp[page, :, :, slot].float()
    hi = p + 1 if s.causal else kv[:, None].expand(-1, Q)
    see = there[:, None] & (j[:, None] < hi[..., None]) & ((j[:, None] < s.sinks) | (j[:, None] > p[..., None] - s.window))
    x = torch.matmul(q.permute(0, 2, 1, 3), k.permute(0, 2, 3, 1)) * SCALE     # [rows, H, Q, N]
    x.masked_fill_(~see[:, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    x = torch.exp(x.sub_(torch.where(m == -math.inf, 0.0, m)))
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x, v.permute(0, 2, 1, 3)) / torch.where(total > 0, total, 1.0)
    o = o.permute(0, 2, 1, 3)[live].to(BF)                            # [n_q, H, 64]
    return o.view(s.q.shape)


def _plain_copy(s):
    src = torch.from_numpy(s.src.astype(np.int64)).to(s.pools[0].device)
    dst = torch.from_numpy(s.dst.astype(np.int64)).to(s.pools[0].device)
    return [p.index_copy_(0, dst, p.index_select(0, src)) for p in s.pools]


def _plain_logprob(s):
    x = s.logits.float()
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    total = e.sum(-1)
    log_total = torch.log(total)
    entropy = log_total - torch.where(e > 0, d * e, 0.0).sum(-1) / total
    lp = d.gather(1, s.tokens[:, None])[:, 0] - log_total
    vals, ids = torch.sort(d, dim=-1, descending=True, stable=True)
    return lp, entropy, vals[:, :s.top] - log_total[:, None], ids[:, :s.top].contiguous()


# --------------------------------------------------------------------------- what a pass cannot do without

def _visible(q, kv, window, sinks, causal):
    """Keys any of the last q queries of a row of kv keys sees, and (query, key) pairs."""
    first = kv - q
    lo = max(0, first - window + 1)
    union = kv - lo + min(sinks, lo) if q else 0
    pairs = 0
    for p in range(first, kv):
        b = max(0, p - window + 1)
        hi = p + 1 if causal else kv
        pairs += hi - b + min(sinks, b)
    return union, pairs


def work(case):
    if case["op"] == "copy":
        page = 2 * case["heads"] * PAGE * HD * 2 * case["layers"]
        return {"bytes": float(page * (case["pairs"] + _sources(case))), "flops": 0.0}
    if case["op"] == "logprob":
        n, k = case["rows"], case["top"]
        size = 4 if case["wide"] else 2
        return {"bytes": float(n * (case["vocab"] * size + 8 + 8 + 12 * k)), "flops": float(n * case["vocab"] * 6)}
    H, rows = case["heads"], case["rows"]
    q_len = _lengths(rows, case["q_lo"], case["q_hi"])
    past = _lengths(rows, case["past_lo"], case["past_hi"])
    # uniform queries or uniform pasts: any pairing of the two has this total
    seen = [_visible(a, a + b, case["window"], case["sinks"], case["causal"]) for a, b in zip(q_len, past)]
    keys, pairs, n_q = sum(u for u, _ in seen), sum(p for _, p in seen), sum(q_len)
    return {"bytes": float(H * HD * 2 * (2 * keys + 2 * n_q) + 4 * (keys // PAGE + 2 * rows)),
            "flops": 4.0 * HD * H * pairs}


# --------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"window": _exact_window, "copy": _exact_copy, "logprob": _exact_logprob}[case["op"]](s)


def _exact_window(s):
    """Row by row: the row's keys laid out densely, a mask of every (query, key), softmax in 64 bits."""
    H = s.pool.shape[2]
    outs, at, q_all = [], 0, s.q.reshape(-1, H, HD).double()
    for r, (n, kv) in enumerate(zip(s.q_host, s.kv_host)):
        npg = (kv + PAGE - 1) // PAGE
        pages = s.pool[s.table[r, :npg].long()]
        K = pages[:, 0].view(npg, H, PAGE, HD).permute(1, 0, 2, 3).reshape(H, npg * PAGE, HD)[:, :kv].double()
        V = pages[:, 1].view(npg, H, HD, PAGE).permute(1, 0, 3, 2).reshape(H, npg * PAGE, HD)[:, :kv].double()
        key = torch.arange(kv, device=K.device)
        for a in range(0, n, 1024):
            b = min(n, a + 1024)
            pos = torch.arange(kv - n + a, kv - n + b, device=K.device)[:, None]
            mask = (key < s.sinks) | (key > pos - s.window)
            if s.causal:
                mask &= key <= pos
            w = torch.einsum("qhd,hkd->hqk", q_all[at + a:at + b], K) * SCALE
            w = torch.softmax(w.masked_fill(~mask, -math.inf), -1)
            outs.append(torch.einsum("hqk,hkd->qhd", w, V))
        at += n
    return torch.cat(outs).view(s.q.shape)


def _exact_copy(s):
    was = [p.clone() for p in s.pools]
    for p, w in zip(s.pools, was):
        for a, b in zip(s.src.tolist(), s.dst.tolist()):
            p[b] = w[a]
    return s.pools


def _exact_logprob(s):
    outs = ([], [], [])
    for a in range(0, s.logits.shape[0], 1024):
        lp = torch.log_softmax(s.logits[a:a + 1024].double(), -1)
        outs[0].append(lp.gather(1, s.tokens[a:a + 1024, None])[:, 0])
        outs[1].append(torch.special.entr(lp.exp()).sum(-1))
        outs[2].append(torch.sort(lp, -1, descending=True)[0][:, :s.top])
    return (*(torch.cat(o) for o in outs), None)
