"""The operators of decoding with drafted tokens, as timed cases: attention for a tree of drafted tokens
over the paged KV cache (bf16 or 8-bit), an 8-bit cache written and read back, the accepted tokens' keys
and values moved together in every layer, and tokens drawn from logits with given random numbers.

Where ``own`` is false, ``run`` computes an operator from elementary torch operations in 32 bits (64 for
sampling, whose borders are sums of many weights); where it is true, it makes the call a user of the
package makes.  ``exact`` is the same result in 64 bits.

Shapes are the T3 backbone's (16 heads of 64, 30 layers, 16-token pages, speech vocabulary 8194) with
generic ones beside them.  Lengths are the mid-quantiles of their distribution, shuffled by the seed:
every seed has other rows but the same total, so ``work`` is exact without the seed.
"""

from __future__ import annotations

import math
import random
from types import SimpleNamespace

import numpy as np
import torch

own = False

PAGE, HD = 16, 64
TILE8 = PAGE * HD + PAGE  # bytes of one head's plane on a page of the 8-bit cache: codes, then scale bytes
SCALE = 0.125
BF = torch.bfloat16
DEV = "cuda"


def listed():
    return [
        # One stream's next token over an 8-bit cache: the smallest call, latency counts.
        dict(name="token8_one", op="tree", rows=1, n_lo=1, n_hi=1, past_lo=1500, past_hi=1500, window=0, sinks=0,
             bits=8, heads=16),
        # A server's single-token step over an 8-bit cache: many streams, very uneven lengths.
        dict(name="token8_batch", op="tree", rows=256, n_lo=1, n_hi=1, past_lo=60, past_hi=4000, window=0, sinks=0,
             bits=8, heads=16),
        # A few requests verify a tree of 24 drafted tokens each, bf16 cache.
        dict(name="draft_few", op="tree", rows=16, n_lo=24, n_hi=24, past_lo=200, past_hi=1500, window=0, sinks=0,
             bits=16, heads=16),
        # Many requests with trees of 1 to 64 tokens, behind a window with sinks, 8-bit cache.
        dict(name="draft8_ragged", op="tree", rows=130, n_lo=1, n_hi=64, past_lo=100, past_hi=3000, window=2000,
             sinks=33, bits=8, heads=16),
        # Three long texts, 13 drafted tokens each: too few rows to fill the chip.
        dict(name="draft_long", op="tree", rows=3, n_lo=13, n_hi=13, past_lo=20000, past_hi=30000, window=0, sinks=0,
             bits=16, heads=16),
        # A step's fresh tokens of a few short rows go into the 8-bit cache, and the rows are read back.
        dict(name="store8_step", op="store", rows=8, n_lo=1, n_hi=1, past_lo=20, past_hi=300, heads=16),
        # Chunks of several prompts on top of what the 8-bit cache has of them, read back for the chunk's attention.
        dict(name="store8_prompts", op="store", rows=37, n_lo=100, n_hi=1500, past_lo=0, past_hi=2500, heads=16),
        # One request's accepted tokens, in every layer.
        dict(name="keep_one", op="keep", rows=1, nodes=24, past_lo=700, past_hi=700, layers=30, bits=16, heads=16),
        # A batch's: most accept a few of 64.
        dict(name="keep_batch", op="keep", rows=130, nodes=64, past_lo=5, past_hi=400, layers=30, bits=16, heads=16),
        # One stream's next token.
        dict(name="sample_one", op="sample", rows=1, vocab=8194, wide=False, masked=False),
        # Every node of 64 requests' trees, some of the vocabulary masked out.
        dict(name="sample_nodes", op="sample", rows=4096, vocab=8194, wide=False, masked=True),
        # A large vocabulary of odd size in fp32.
        dict(name="sample_wide", op="sample", rows=300, vocab=100003, wide=True, masked=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["token", "token", "draft", "draft", "store", "keep", "sample", "sample"])
    heads = rng.choice([4, 8, 16, 16])
    if op in ("token", "draft"):
        rows = _log_int(rng, 1, 250 if op == "token" else 120)
        lo = _log_int(rng, 1, 3000)
        hi = min(lo * rng.randint(1, 8), 12000, max(lo, 400000 // rows))
        n_hi = 1 if op == "token" else rng.randint(2, 64)
        n_lo = n_hi if rng.choice([True, False]) else rng.randint(1, n_hi)
        windowed = rng.choice([False, False, True])
        return dict(op="tree", rows=rows, n_lo=n_lo, n_hi=n_hi, past_lo=lo, past_hi=hi,
                    window=_log_int(rng, 65, 3000) if windowed else 0,
                    sinks=rng.choice([0, 1, 4, 31, 64]) if windowed else 0, bits=rng.choice([16, 8, 8]), heads=heads)
    if op == "store":
        rows = _log_int(rng, 1, 100)
        hi = _log_int(rng, 1, max(1, 40000 // rows))
        past = rng.choice([0, _log_int(rng, 1, max(1, 60000 // rows))])
        return dict(op="store", rows=rows, n_lo=rng.choice([1, hi]), n_hi=hi, past_lo=rng.randint(0, past), past_hi=past,
                    heads=heads)
    if op == "keep":
        past = rng.randint(0, 600)
        return dict(op="keep", rows=_log_int(rng, 1, 100), nodes=rng.randint(2, 64), past_lo=rng.randint(0, past),
                    past_hi=past, layers=rng.choice([1, 12, 30]), bits=rng.choice([16, 8]), heads=heads)
    wide = rng.choice([False, False, True])
    vocab = rng.choice([8194, 8194, _log_int(rng, 50, 120000)])
    rows = _log_int(rng, 1, min(4096, 30 * 1000 * 1000 // vocab))
    return dict(op="sample", rows=rows, vocab=vocab, wide=wide, masked=rng.choice([False, True]))


# --------------------------------------------------------------------------- inputs

def _lengths(n, lo, hi, seed=None):
    """n lengths in [lo, hi] at the mid-quantiles of a uniform distribution, shuffled by the seed."""
    out = [int(round(lo + (hi - lo) * (i + 0.5) / n)) for i in range(n)]
    if seed is not None:
        random.Random(seed).shuffle(out)
    return out


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _starts(lengths):
    out = [0]
    for x in lengths:
        out.append(out[-1] + x)
    return out


def _table(lengths, seed):
    """Pages of rows of these lengths in a shuffled pool: (table on the host, pages of the pool)."""
    pages = [(x + PAGE - 1) // PAGE for x in lengths]
    n_pages = sum(lengths) // PAGE + len(lengths) + 8  # enough for every order of the lengths
    order = np.random.default_rng(seed).permutation(n_pages).astype(np.int32)
    table, at = np.zeros((len(lengths), max(max(pages), 1)), dtype=np.int32), 0
    for r, n in enumerate(pages):
        table[r, :n] = order[at:at + n]
        at += n
    return table, n_pages


def _pool(g, n_pages, heads, bits):
    if bits == 16:
        return torch.empty(n_pages, 2, heads, PAGE * HD, dtype=BF, device=DEV).normal_(generator=g)
    # codes of normal vectors: the largest of 64 values is near 100 of 127 at these scales
    pool = torch.empty(n_pages, 2, heads, TILE8, dtype=torch.uint8, device=DEV)
    codes = torch.empty(n_pages, 2, heads, PAGE * HD, device=DEV).normal_(std=36.0, generator=g)
    pool[..., :PAGE * HD] = codes.round_().clamp_(-127, 127).to(torch.int8).view(torch.uint8)
    pool[..., PAGE * HD:] = torch.randint(121, 124, (n_pages, 2, heads, PAGE), generator=g, device=DEV).to(torch.uint8)
    return pool


def prepare(case, seed):
    return {"tree": _prepare_tree, "store": _prepare_store, "keep": _prepare_keep, "sample": _prepare_sample}[case["op"]](
        case, seed)


def _trees(q_len, seed):
    """A drafted tree for every row: each node's parent is an earlier node of the row or the row's last token
    (none).  The masks name a node's ancestors and itself."""
    rng = np.random.default_rng(seed)
    masks = []
    for n in q_len:
        row = []
        for i in range(n):
            parent = int(rng.integers(-1, i)) if i else -1
            row.append((row[parent] if parent >= 0 else 0) | 1 << i)
        masks += row
    return np.array(masks, dtype=np.uint64).view(np.int64)


def _prepare_tree(case, seed):
    g, H, rows = _gen(seed), case["heads"], case["rows"]
    q_len = _lengths(rows, case["n_lo"], case["n_hi"], seed)
    past = _lengths(rows, case["past_lo"], case["past_hi"], seed + 1)
    kv_len = [a + b for a, b in zip(past, q_len)]
    table, n_pages = _table(kv_len, seed)
    packed = case["n_lo"] != case["n_hi"]
    mask = torch.from_numpy(_trees(q_len, seed)).to(DEV)
    # queries with some spread, so that a softmax has weight on a few keys
    q = (torch.randn(sum(q_len), H, HD, generator=g, device=DEV) * 2).to(BF)
    shape = (-1,) if packed else (rows, case["n_hi"])
    return SimpleNamespace(op="tree", q=q.view(*shape, H, HD), mask=mask.view(shape), packed=packed,
                           pool=_pool(g, n_pages, H, case["bits"]), table=torch.from_numpy(table).to(DEV),
                           kv_len=_ints(kv_len), q_start=_ints(_starts(q_len)), max_q=max(q_len), max_kv=max(kv_len),
                           window=case["window"] or None, sinks=case["sinks"], kv_host=kv_len, q_host=q_len)


def _prepare_store(case, seed):
    g, H, rows = _gen(seed), case["heads"], case["rows"]
    n_new = _lengths(rows, case["n_lo"], case["n_hi"], seed)
    past = _lengths(rows, case["past_lo"], case["past_hi"], seed + 1)
    kv_len = [a + b for a, b in zip(past, n_new)]
    table, n_pages = _table(kv_len, seed)
    wide_table, n_wide = _table(kv_len, seed + 1)
    # keys and values as the projections leave them: slices of one buffer; a few channels much larger
    n = sum(n_new)
    qkv = torch.randn(n, 3, H, HD, generator=g, device=DEV)
    qkv[..., 5] *= 8
    qkv = qkv.to(BF)
    return SimpleNamespace(op="store", k=qkv[:, 1], v=qkv[:, 2], pool8=_pool(g, n_pages, H, 8),
                           table=torch.from_numpy(table).to(DEV), pos0=_ints(past), kv_len=_ints(kv_len),
                           q_start=_ints(_starts(n_new)), max_kv=max(kv_len),
                           pool=torch.zeros(n_wide, 2, H, PAGE * HD, dtype=BF, device=DEV),
                           wide_table=torch.from_numpy(wide_table).to(DEV))


def _n_kept(case):
    """How many nodes each row keeps: from none to a third of its tree (16 at most), more of the small counts."""
    top = min(max(case["nodes"] // 3, 1), 16)
    rows = case["rows"]
    return [int(round(top * ((i + 0.5) / rows) ** 2)) for i in range(rows)] if rows > 1 else [max(1, top // 2)]


def _prepare_keep(case, seed):
    g, rows, nodes = _gen(seed), case["rows"], case["nodes"]
    base = _lengths(rows, case["past_lo"], case["past_hi"], seed)
    table, n_pages = _table([b + nodes for b in base], seed)
    n_kept = _n_kept(case)
    random.Random(seed).shuffle(n_kept)
    rng = np.random.default_rng(seed)
    kept = np.zeros((rows, nodes), dtype=np.int32)
    for r, m in enumerate(n_kept):
        kept[r, :m] = np.sort(rng.choice(nodes, m, replace=False))
    return SimpleNamespace(op="keep", pools=[_pool(g, n_pages, case["heads"], case["bits"]) for _ in range(case["layers"])],
                           table=torch.from_numpy(table).to(DEV), base=_ints(base), kept=torch.from_numpy(kept).to(DEV),
                           n_kept=_ints(n_kept))


def _prepare_sample(case, seed):
    g, rows, V = _gen(seed), case["rows"], case["vocab"]
    pitch = (V + 7) // 8 * 8  # rows as the speech head leaves them: padded to 16 bytes
    x = torch.empty(rows, pitch, dtype=torch.float32 if case["wide"] else BF, device=DEV)
    logits = x.normal_(std=3.0, generator=g)[:, :V]
    if case["masked"]:  # an eighth of the vocabulary is not allowed, the first token always
        off = torch.rand(V, generator=g, device=DEV) < 0.125
        off[0] = False
        logits[:, off] = -math.inf

    def of(values, dtype):  # every request has settings of its own
        at = torch.randint(0, len(values), (rows,), generator=g, device=DEV)
        return torch.tensor(values, dtype=dtype, device=DEV)[at]

    return SimpleNamespace(op="sample", logits=logits, u=torch.rand(rows, generator=g, device=DEV),
                           temperature=of([0.0, 0.6, 0.8, 0.8, 1.0, 1.3], torch.float32),
                           top_k=of([0, 0, 1, 20, 50, 1000], torch.int32),
                           top_p=of([1.0, 1.0, 0.8, 0.9, 0.95], torch.float32),
                           min_p=of([0.0, 0.0, 0.02, 0.05], torch.float32))


# --------------------------------------------------------------------------- one pass

def run(state):
    if own:
        return {"tree": _own_tree, "store": _own_store, "keep": _own_keep, "sample": _own_sample}[state.op](state)
    return {"tree": _plain_tree, "store": _plain_store, "keep": _plain_keep, "sample": _plain_sample}[state.op](state)


def _own_tree(s):
    from yapd_amd import kernels
    out = torch.empty_like(s.q)
    kernels.attn_tree(s.q, s.pool, s.table, s.kv_len, s.mask, out, SCALE, window=s.window, sinks=s.sinks,
                      q_start=s.q_start if s.packed else None, max_q=s.max_q, max_kv=s.max_kv)
    return out


def _own_store(s):
    from yapd_amd import kernels
    kernels.kv8_write(s.k, s.v, s.pool8, s.table, s.pos0, q_start=s.q_start)
    kernels.kv8_unpack(s.pool8, s.table, s.kv_len, s.pool, s.wide_table, max_kv=s.max_kv)
    return s.pool


def _own_keep(s):
    from yapd_amd import kernels
    kernels.kv_keep(s.pools, s.table, s.base, s.kept, s.n_kept)
    return s.pools


def _own_sample(s):
    from yapd_amd import scoring
    r = scoring.sample_tokens(s.logits, s.u, temperature=s.temperature, top_k=s.top_k, top_p=s.top_p, min_p=s.min_p)
    return r.token, r.logprob


def _power(byte):
    """2^(byte - 127) in 32 bits: the byte is the exponent's."""
    return (byte.to(torch.int32) << 23).view(torch.float32)


def _keys_values(pool, page, slot):
    """K and V in 32 bits at (page, slot) index tensors of one shape: [..., H, 64] each."""
    H = pool.shape[2]
    if pool.dtype == BF:
        k = pool[:, 0].view(-1, H, PAGE, HD)[page, :, slot].float()
        return k, pool[:, 1].view(-1, H, HD, PAGE)[page, :, :, slot].float()
    codes, scale = pool[..., :PAGE * HD].view(torch.int8), _power(pool[..., PAGE * HD:])  # [pages, 2, H, 1024 and 16]
    k = codes[:, 0].reshape(-1, H, PAGE, HD)[page, :, slot].float() * scale[:, 0][page, :, slot][..., None]
    return k, codes[:, 1].reshape(-1, H, HD, PAGE)[page, :, :, slot].float() * scale[:, 1][page, :, slot][..., None]


def _plain_tree(s):
    """Every row's keys gathered from the pages (behind the window where there is one), one masked softmax."""
    H, rows, Q, dev = s.pool.shape[2], s.kv_len.numel(), s.max_q, s.pool.device
    kv, start = s.kv_len.long(), s.q_start.long()
    n = start[1:] - start[:-1]
    i = torch.arange(Q, device=dev)
    live = i[None, :] < n[:, None]                                    # [rows, Q]
    at = (start[:-1, None] + i).clamp_max(s.q.numel() // (H * HD) - 1)
    q = s.q.reshape(-1, H, HD)[at].float()
    mask = s.mask.reshape(-1)[at]                                     # [rows, Q]
    ctx = kv - n
    bit = (mask[..., None] >> torch.arange(64, device=dev)) & 1       # [rows, Q, 64]
    depth = bit.sum(-1) - torch.gather(bit, 2, i[None, :, None].expand(rows, Q, 1))[..., 0]
    window = s.window or s.max_kv + 64
    first = (ctx - window + 1).clamp_min(s.sinks)                     # first key behind the sinks
    span = min(s.max_kv, window + Q)
    sink = torch.arange(s.sinks, device=dev).expand(rows, -1)
    j = torch.cat([sink, first[:, None] + torch.arange(span, device=dev)], 1)  # [rows, N] key positions
    there = j < kv[:, None]
    jc = torch.where(there, j, 0)
    k, v = _keys_values(s.pool, torch.gather(s.table.long(), 1, jc // PAGE), jc % PAGE)
    node = j - ctx[:, None]                                           # a key's node, below 0 in the context
    own_bit = torch.gather(bit, 2, node.clamp(0, 63)[:, None, :].expand(-1, Q, -1)) == 1
    p = ctx[:, None] + depth
    near = (j < s.sinks)[:, None] | (j[:, None] > p[..., None] - window)
    see = there[:, None] & torch.where((node < 0)[:, None], near, own_bit)
    x = torch.matmul(q.permute(0, 2, 1, 3), k.permute(0, 2, 3, 1)) * SCALE     # [rows, H, Q, N]
    x.masked_fill_(~see[:, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    x = torch.exp(x.sub_(torch.where(m == -math.inf, 0.0, m)))
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x, v.permute(0, 2, 1, 3)) / torch.where(total > 0, total, 1.0)
    return o.permute(0, 2, 1, 3)[live].to(BF).view(s.q.shape)


def _plain_store(s):
    H = s.pool8.shape[2]
    n = (s.q_start[1:] - s.q_start[:-1]).long()
    rows = torch.repeat_interleave(torch.arange(n.numel(), device=s.k.device), n, output_size=s.k.shape[0])
    pos = s.pos0.long()[rows] + torch.arange(s.k.shape[0], device=s.k.device) - s.q_start.long()[rows]
    page, slot = s.table.long()[rows, pos // PAGE], pos % PAGE
    for plane, x in ((0, s.k.float()), (1, s.v.float())):
        e = (torch.frexp(x.abs().amax(-1)).exponent - 7).clamp_min(-126)       # [tokens, H]
        c = (x / _power(e + 127)[..., None]).round().clamp(-127, 127).to(torch.int8).view(torch.uint8)
        tile = s.pool8[:, plane]                                               # [pages, H, 1040]
        d = torch.arange(HD, device=x.device)
        h = torch.arange(H, device=x.device)
        where = slot[:, None] * HD + d if plane == 0 else d * PAGE + slot[:, None]  # [tokens, 64]
        tile[page[:, None, None], h[:, None], where[:, None, :]] = c
        tile[page[:, None], h, PAGE * HD + slot[:, None]] = (e + 127).to(torch.uint8)
    cols = torch.arange(s.table.shape[1], device=s.k.device)
    used = cols[None, :] * PAGE < s.kv_len[:, None]
    src, dst = s.table[used].long(), s.wide_table[used].long()
    t = s.pool8[src]
    scale = _power(t[..., PAGE * HD:])                                         # [n, 2, H, 16]
    c = t[..., :PAGE * HD].contiguous().view(torch.int8).float()
    s.pool[dst, 0] = (c[:, 0].view(-1, H, PAGE, HD) * scale[:, 0][..., None]).to(BF).view(-1, H, PAGE * HD)
    s.pool[dst, 1] = (c[:, 1].view(-1, H, HD, PAGE) * scale[:, 1][:, :, None]).to(BF).view(-1, H, PAGE * HD)
    return s.pool


def _plain_keep(s):
    m = s.kept.shape[1]
    take = torch.arange(m, device=s.kept.device)[None, :] < s.n_kept[:, None]
    r, i = take.nonzero(as_tuple=True)
    old, new = s.base.long()[r] + s.kept[r, i], s.base.long()[r] + i
    table = s.table.long()
    op, os, np_, ns = table[r, old // PAGE], old % PAGE, table[r, new // PAGE], new % PAGE
    for pool in s.pools:
        H = pool.shape[2]
        codes = pool[..., :PAGE * HD]
        k, v = codes[:, 0].unflatten(-1, (PAGE, HD)), codes[:, 1].unflatten(-1, (HD, PAGE))
        k_old, v_old = k[op, :, os], v[op, :, :, os]
        scales = None
        if pool.dtype == torch.uint8:
            scales = pool[..., PAGE * HD:]
            s_old = scales[op, :, :, os]
        h, d = torch.arange(H, device=r.device), torch.arange(HD, device=r.device)
        k[np_[:, None], h, ns[:, None]] = k_old
        v[np_[:, None, None], h[:, None], d, ns[:, None, None]] = v_old
        if scales is not None:
            scales[np_[:, None, None], torch.arange(2, device=r.device)[:, None], h, ns[:, None, None]] = s_old
    return s.pools


def _plain_sample(s):
    x = s.logits.double()
    V = x.shape[1]
    x, order = torch.sort(x, dim=-1, descending=True, stable=True)
    t = s.temperature.double()[:, None]
    w = torch.exp((x - x[:, :1]) / torch.where(t > 0, t, 1.0))
    total = torch.cumsum(w, -1)
    rank = torch.arange(V, device=x.device)
    k = torch.where((s.top_k <= 0) | (s.top_k > V), V, s.top_k).long()[:, None]
    k = torch.where(t > 0, k, 1)
    z = total.gather(1, k - 1)
    before = torch.cat([torch.zeros_like(z), total[:, :-1]], 1)
    keep = (rank < k) & ((rank == 0) | (before < s.top_p.double()[:, None] * z) | (s.top_p >= 1)[:, None])
    keep &= (rank == 0) | (w >= s.min_p.double()[:, None])
    z = total.gather(1, keep.sum(-1, keepdim=True) - 1)
    at = (total <= s.u.double()[:, None] * z).sum(-1, keepdim=True)
    return order.gather(1, at)[:, 0], torch.log(w.gather(1, at) / z)[:, 0].float()


# --------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    H, rows = case["heads"] if "heads" in case else 0, case["rows"]
    if case["op"] == "sample":
        n = rows * case["vocab"]
        return {"bytes": float(n * (4 if case["wide"] else 2) + rows * 32), "flops": float(n * 6)}
    if case["op"] == "keep":
        tokens = sum(_n_kept(case))
        return {"bytes": float(tokens * case["layers"] * H * 2 * (256 if case["bits"] == 16 else 130)), "flops": 0.0}
    new = _lengths(rows, case["n_lo"], case["n_hi"])
    past = _lengths(rows, case["past_lo"], case["past_hi"])
    if case["op"] == "store":
        # the fresh tokens' K and V and their codes, then the earlier tokens' codes and every token's values
        return {"bytes": float(H * (sum(new) * (256 + 130) + sum(past) * 130 + (sum(new) + sum(past)) * 256)),
                "flops": float(H * 128 * (sum(new) * 3 + sum(past)))}
    keys = pairs = 0
    for n, ctx in zip(new, past):  # uniform trees or any pairing of the two: close to every seed's total
        seen = min(ctx, case["window"] - 1) if case["window"] else ctx
        seen += min(case["sinks"], ctx - seen)
        keys += seen + n
        pairs += n * (seen + 1)
    byte = 256 if case["bits"] == 16 else 130
    return {"bytes": float(H * (keys * byte + sum(new) * 256) + 4 * (keys // PAGE + 2 * rows) + 8 * sum(new)),
            "flops": 4.0 * HD * H * pairs}


# --------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"tree": _exact_tree, "store": _exact_store, "keep": _exact_keep, "sample": _exact_sample}[case["op"]](s)


def _dense(pool, pages, plane):
    """One plane of a row's pages as [H, tokens, 64] in 64 bits."""
    t, H = pool[pages, plane], pool.shape[2]
    scale = None
    if pool.dtype == torch.uint8:
        powers = torch.tensor([math.ldexp(1.0, i - 127) for i in range(256)], dtype=torch.float64, device=t.device)
        scale = powers[t[..., PAGE * HD:].long()].permute(1, 0, 2).reshape(H, -1, 1)
        t = t[..., :PAGE * HD].contiguous().view(torch.int8)
    t = t.double()
    t = t.view(-1, H, PAGE, HD).permute(1, 0, 2, 3) if plane == 0 else t.view(-1, H, HD, PAGE).permute(1, 0, 3, 2)
    t = t.reshape(H, -1, HD)
    return t if scale is None else t * scale


def _exact_tree(s):
    """Row by row: the row's keys laid out densely, the mask of every (node, key) from the tree's bits."""
    H = s.pool.shape[2]
    q_all, masks = s.q.reshape(-1, H, HD).double(), s.mask.reshape(-1).cpu().numpy().view(np.uint64)
    outs, at = [], 0
    for r, (n, kv) in enumerate(zip(s.q_host, s.kv_host)):
        pages = s.table[r, :(kv + PAGE - 1) // PAGE].long()
        K, V = _dense(s.pool, pages, 0)[:, :kv], _dense(s.pool, pages, 1)[:, :kv]
        see = np.zeros((n, kv), dtype=bool)
        for i in range(n):
            bits = int(masks[at + i])
            depth = bin(bits & ~(1 << i)).count("1")
            lo = max(0, kv - n + depth - s.window + 1) if s.window else 0
            see[i, lo:kv - n] = True
            see[i, :min(s.sinks, kv - n)] = True
            see[i, kv - n:] = [bool(bits >> j & 1) for j in range(n)]
        w = torch.einsum("qhd,hkd->hqk", q_all[at:at + n], K) * SCALE
        w = torch.softmax(w.masked_fill(~torch.from_numpy(see).to(w.device), -math.inf), -1)
        outs.append(torch.einsum("hqk,hkd->qhd", w, V))
        at += n
    return torch.cat(outs).view(s.q.shape)


def _exact_store(s):
    """Row by row: the row's vectors before and after the fresh ones are rounded to 127 steps a side."""
    H, out = s.pool8.shape[2], s.pool.double()
    start, pos0, kv_len = s.q_start.tolist(), s.pos0.tolist(), s.kv_len.tolist()
    for r, kv in enumerate(kv_len):
        cols = (kv + PAGE - 1) // PAGE
        src, dst = s.table[r, :cols].long(), s.wide_table[r, :cols].long()
        for plane, x in ((0, s.k), (1, s.v)):
            dense = _dense(s.pool8, src, plane)                                # [H, cols * 16, 64]
            new = x[start[r]:start[r + 1]].double()
            top = new.abs().amax(-1, keepdim=True).cpu().numpy()
            step = torch.from_numpy(np.ldexp(1.0, np.maximum(np.frexp(top)[1] - 7, -126))).to(new.device)
            dense[:, pos0[r]:kv] = ((new / step).round().clamp(-127, 127) * step).permute(1, 0, 2)
            tiles = dense.view(H, cols, PAGE, HD).permute(1, 0, 2, 3)
            out[dst, plane] = (tiles if plane == 0 else tiles.transpose(2, 3)).reshape(cols, H, PAGE * HD)
    return out


def _exact_keep(s):
    base, n_kept, kept, table = s.base.tolist(), s.n_kept.tolist(), s.kept.tolist(), s.table.tolist()
    for pool in s.pools:
        was = pool.clone()
        for r in range(len(base)):
            for i in range(n_kept[r]):
                a, b = base[r] + kept[r][i], base[r] + i
                pa, pb, sa, sb = table[r][a // PAGE], table[r][b // PAGE], a % PAGE, b % PAGE
                pool[pb, 0, :, sb * HD:sb * HD + HD] = was[pa, 0, :, sa * HD:sa * HD + HD]
                pool[pb, 1, :, sb:PAGE * HD:PAGE] = was[pa, 1, :, sa:PAGE * HD:PAGE]
                if pool.dtype == torch.uint8:
                    pool[pb, :, :, PAGE * HD + sb] = was[pa, :, :, PAGE * HD + sa]
    return s.pools


def _exact_sample(s):
    """Row by row on the host: the weights in order, the three prefixes, and the place of u in the shortest."""
    x_all = s.logits.double().cpu().numpy()
    setting = [v.cpu().numpy().astype(np.float64) for v in (s.temperature, s.top_k, s.top_p, s.min_p, s.u)]
    tokens, logprobs = [], []
    for x, T, k, p, m, u in zip(x_all, *setting):
        order = np.argsort(-x, kind="stable")
        if T == 0:
            tokens.append(int(order[0]))
            logprobs.append(0.0)
            continue
        w = np.exp((x[order] - x[order[0]]) / T)
        if 0 < k < len(w):
            w = w[:int(k)]
        if p < 1:
            w = w[:max(1, int(np.searchsorted(np.cumsum(w), p * w.sum(), side="left")) + 1)]
        w = w[:max(1, int(np.count_nonzero(w >= m)))]
        c = np.cumsum(w)
        at = int(np.searchsorted(c, u * c[-1], side="right"))
        tokens.append(int(order[at]))
        logprobs.append(math.log(w[at] / c[-1]))
    dev = s.logits.device
    return torch.tensor(tokens, device=dev), torch.tensor(logprobs, dtype=torch.float64, device=dev)
