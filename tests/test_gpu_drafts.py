"""GPU: decoding with drafted trees, its pieces used together: a cache of either width with pages mapped on demand, the trees'
keys written, attention over them, tokens drawn for every node, the accepted path kept, pages behind a window given back."""

import numpy as np
import pytest
import torch

from oracle import kv8 as OK
from oracle import sample as OS
from oracle import tree as OT
from oracle import window as OW
from tests._tree_cases import tolerance
from yapd_amd import kernels, scoring
from yapd_amd.paged import PagedKV, SharedPagedKV

pytestmark = pytest.mark.gpu

H, LAYERS, VOCAB, SCALE = 4, 2, 97, 0.125
PARENTS = [-1, 0, 0, 1, 1, 2, 3, 6]
DEPTH = [0, 1, 1, 2, 2, 2, 3, 4]


class World:
    """Queries, keys and values are functions of (token, position); the next token's logits are a bias of the token
    plus the attention's output through a head.  The bias is the larger part, so that a rounding never decides."""

    def __init__(self, dev, bits, window, sinks, n_rows=3):
        g = torch.Generator().manual_seed(11)
        r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        self.dev, self.bits, self.window, self.sinks = dev, bits, window, sinks
        self.tok = [[r(VOCAB, H, 64) for _ in range(3)] for _ in range(LAYERS)]
        self.pos = [[r(512, H, 64) for _ in range(3)] for _ in range(LAYERS)]
        self.bias = 4 * r(VOCAB, VOCAB)
        self.head = 0.02 * r(LAYERS * H * 64, VOCAB)
        self.u = torch.rand(n_rows, 512, generator=g)
        self.kv = SharedPagedKV(n_layers=LAYERS, n_rows=n_rows, pages_per_row=16, n_heads=H, device=dev, n_pages=40, kv_bits=bits)
        self.rng = np.random.default_rng(5)

    def qkv(self, layer, which, tokens, positions):
        return (self.tok[layer][which][tokens] + self.pos[layer][which][positions]).bfloat16()

    def value(self, x):
        """What the cache holds of a vector."""
        return OK.values(*OK.quantise(x)) if self.bits == 8 else x.double()

    def logits(self, tokens, outs):
        """bf16 logits of tokens whose attention outputs (per layer, [n, H, 64]) are given."""
        hidden = torch.cat([o.double().reshape(len(tokens), -1) for o in outs], 1)
        return (self.bias[tokens].double() + hidden @ self.head.double()).bfloat16()

    def next_token(self, row, position, logits, T):
        return OS.sample_row(logits.double().numpy(), float(self.u[row, position]), T, 20, 0.9, 0.02)[0]

    def one_by_one(self, row, prompt, n, T):
        """The row's next n tokens, each from attention in 64 bits over everything before."""
        tokens = list(prompt)
        for _ in range(n):
            p = len(tokens) - 1
            outs = []
            for layer in range(LAYERS):
                t, at = torch.tensor(tokens), torch.arange(p + 1)
                K, V = (self.value(self.qkv(layer, w, t, at)) for w in (1, 2))
                see = OT.visible(p + 1, 1, [1], self.window, self.sinks)
                outs.append(OT.attend(self.qkv(layer, 0, t[-1:], at[-1:]), K, V, see, SCALE)[0])
            tokens.append(self.next_token(row, p + 1, self.logits(tokens[-1:], outs)[0], T))
        return tokens[len(prompt):]

    def write(self, layer, rows_tokens, rows_positions, pos0, n):
        """Keys and values of n tokens a row to slots pos0[r] and on, in every row of the cache."""
        t, at = torch.tensor(rows_tokens).view(-1), torch.tensor(rows_positions).view(-1)
        k, v = (self.qkv(layer, w, t, at).to(self.dev) for w in (1, 2))
        p0 = torch.tensor(pos0, dtype=torch.int32, device=self.dev)
        if self.bits == 8:
            kernels.kv8_write(k, v, self.kv.pools[layer], self.kv.table, p0)
        else:
            kernels.kv_write(k, v, self.kv.pools[layer], self.kv.table, p0, n)


@pytest.mark.parametrize("T", [0.0, 0.7])
@pytest.mark.parametrize("bits,window,sinks", [(16, None, 0), (8, None, 0), (8, 40, 5)])
def test_drafts_give_the_tokens_of_decoding_one_by_one(dev, bits, window, sinks, T):
    w = World(dev, bits, window, sinks)
    rows, n, rounds = 3, len(PARENTS), 14
    prompt = [[int(x) for x in w.rng.integers(0, VOCAB, 33)] for _ in range(rows)]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    for r in range(rows):
        w.kv.reserve(r, 0, 32)
    for layer in range(LAYERS):
        w.write(layer, [p[:32] for p in prompt], [list(range(32))] * rows, [0] * rows, 32)
    tokens = [list(p) for p in prompt]  # the last one is not in the cache yet
    masks = torch.from_numpy(kernels.tree_masks(PARENTS)).to(dev).expand(rows, n).contiguous()
    taken = 0
    want = [w.one_by_one(r, prompt[r], rounds * 5, T) for r in range(rows)]
    for _ in range(rounds):
        base = [len(t) - 1 for t in tokens]
        drafts = []
        for r in range(rows):  # the first child often is the right token, as a good draft's
            row = [tokens[r][-1]]
            for i in range(1, n):
                right = want[r][base[r] + DEPTH[i] - 33] if base[r] + DEPTH[i] - 33 < len(want[r]) else 0
                row.append(right if PARENTS.index(PARENTS[i]) == i and w.rng.random() < 0.8 else int(w.rng.integers(0, VOCAB)))
            drafts.append(row)
            w.kv.reserve(r, base[r], base[r] + n)
        positions = [[b + d for d in DEPTH] for b in base]
        outs, kv_len = [], i32([b + n for b in base])
        for layer in range(LAYERS):
            w.write(layer, drafts, positions, base, n)
            q = w.qkv(layer, 0, torch.tensor(drafts).view(-1), torch.tensor(positions).view(-1)).to(dev).view(rows, n, H, 64)
            out = torch.full_like(q, 77.0)
            kernels.attn_tree(q, w.kv.pools[layer], w.kv.table, kv_len, masks, out, SCALE, window=window, sinks=sinks)
            outs.append(out.cpu())
        logits = torch.stack([w.logits(drafts[r], [o[r] for o in outs]) for r in range(rows)]).to(dev)
        u = torch.stack([w.u[r, [p + 1 for p in positions[r]]] for r in range(rows)]).to(dev)
        drawn = scoring.sample_tokens(logits, u, temperature=T, top_k=20, top_p=0.9, min_p=0.02).token.cpu()
        kept = np.zeros((rows, n), dtype=np.int32)
        count = []
        for r in range(rows):
            path = [0]
            while True:
                token = int(drawn[r, path[-1]])
                tokens[r].append(token)
                child = [i for i in range(n) if PARENTS[i] == path[-1] and drafts[r][i] == token]
                if not child:
                    break
                path.append(child[0])
            kept[r, :len(path)] = path
            count.append(len(path))
        taken += sum(count)
        w.kv.keep_nodes(i32(base), torch.from_numpy(kept).to(dev), i32(count))
        for r in range(rows):
            if window:
                w.kv.release_before(r, len(tokens[r]) - window, sinks)
    for r in range(rows):
        got = tokens[r][33:]
        assert len(got) >= rounds and got == want[r][:len(got)]
    assert taken > rounds * rows * 1.5, "drafts were hardly ever accepted"
    # what is left in the cache is what decoding one by one would have written
    torch.cuda.synchronize()
    for layer, pool in enumerate(p.cpu() for p in w.kv.pools):
        for r in range(rows):
            t, at = torch.tensor(tokens[r][:-1]), torch.arange(len(tokens[r]) - 1)
            for plane in (0, 1):
                x = w.value(w.qkv(layer, 1 + plane, t, at))
                for p in range(len(t)):
                    page = int(w.kv.table_host[r, p // 16])
                    if page == 0:
                        assert window and sinks <= p < len(tokens[r]) - window
                        continue
                    if bits == 8:
                        got = OK.read(pool, page, p % 16, plane)
                    else:
                        tile = pool[page, plane].double()
                        got = tile.view(H, 16, 64)[:, p % 16] if plane == 0 else tile.view(H, 64, 16)[:, :, p % 16]
                    assert torch.equal(got, x[p]), (layer, r, plane, p)


def test_a_chunk_of_a_prompt_on_an_8_bit_cache(dev):
    """Chunks longer than a tree: written to the 8-bit cache, read back into pages that the windowed attention reads."""
    w = World(dev, 8, 60, 3, n_rows=2)
    wide = PagedKV(n_layers=1, n_rows=2, pages_per_row=16, n_heads=H, device=dev, shuffle_seed=4)
    g = torch.Generator().manual_seed(2)
    length = [0, 0]
    dense = [[[], []], [[], []]]
    for lens in ([70, 5], [90, 101], [1, 80]):
        k, v, q = ((2 * torch.randn(sum(lens), H, 64, generator=g)).bfloat16() for _ in range(3))
        start = torch.tensor([0, lens[0], sum(lens)], dtype=torch.int32, device=dev)
        for r in range(2):
            w.kv.reserve(r, length[r], length[r] + lens[r])
        kernels.kv8_write(k.to(dev), v.to(dev), w.kv.pools[0], w.kv.table,
                          torch.tensor(length, dtype=torch.int32, device=dev), q_start=start)
        length = [a + b for a, b in zip(length, lens)]
        kv_len = torch.tensor(length, dtype=torch.int32, device=dev)
        kernels.kv8_unpack(w.kv.pools[0], w.kv.table, kv_len, wide.pools[0], wide.table)
        out = torch.full_like(q, 77.0, device=dev)
        kernels.attn_window(q.to(dev), wide.pools[0], wide.table, kv_len, out, SCALE, window=60, sinks=3, q_start=start)
        out = out.cpu().double()
        for r in range(2):
            s = slice(0, lens[0]) if r == 0 else slice(lens[0], sum(lens))
            for i, x in enumerate((k, v)):
                dense[r][i].append(OK.values(*OK.quantise(x[s])))
            want, a = OW.attend(q[s], torch.cat(dense[r][0]), torch.cat(dense[r][1]), 60, 3, True, SCALE)
            # the tile kernel of long chunks rounds its weights against a maximum that may lag: twice the bound
            assert bool(((out[s] - want).abs() <= 2 * tolerance(want, a)).all()), (r, lens)


@pytest.mark.parametrize("bits", [16, 8])
def test_a_captured_round_follows_its_buffers(dev, bits):
    """Write, attention, sampling and keeping in one graph, replayed on other nodes, lengths, masks and numbers, against
    the same calls made one after the other."""
    rows, n, cols = 3, 9, 8
    kv = PagedKV(n_layers=2, n_rows=rows, pages_per_row=cols, n_heads=H, device=dev, shuffle_seed=1, kv_bits=bits)
    rng = np.random.default_rng(0)
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt, device=dev)  # noqa: E731
    b = dict(q=z(rows, n, H, 64), k=z(rows * n, H, 64), v=z(rows * n, H, 64), mask=z(rows, n, dt=torch.int64),
             base=z(rows, dt=torch.int32), kv_len=z(rows, dt=torch.int32), kept=z(rows, n, dt=torch.int32),
             count=z(rows, dt=torch.int32), logits=z(rows, n, 130), u=z(rows, n, dt=torch.float32))
    out, token, lp = z(rows, n, H, 64), z(rows, n, dt=torch.int64), z(rows, n, dt=torch.float32)

    def call():
        for pool in kv.pools:
            if bits == 8:
                kernels.kv8_write(b["k"], b["v"], pool, kv.table, b["base"])
            else:
                kernels.kv_write(b["k"], b["v"], pool, kv.table, b["base"], n)
        kernels.attn_tree(b["q"], kv.pools[1], kv.table, b["kv_len"], b["mask"], out, SCALE)
        kernels.sample_tokens(b["logits"], b["u"], token, lp, temperature=0.9, top_p=0.8)
        kernels.kv_keep(kv.pools, kv.table, b["base"], b["kept"], b["count"])

    def fill(seed):
        g = torch.Generator().manual_seed(seed)
        for name in ("q", "k", "v", "logits"):
            b[name].copy_(2 * torch.randn(b[name].shape, generator=g))
        b["u"].copy_(torch.rand(rows, n, generator=g))
        base = torch.randint(0, cols * 16 - n + 1, (rows,), generator=g)
        b["base"].copy_(base)
        b["kv_len"].copy_(base + n)
        b["mask"].copy_(torch.stack([torch.from_numpy(kernels.tree_masks([-1] + [int(rng.integers(-1, i)) for i in range(1, n)]))
                                     for _ in range(rows)]))
        b["kept"].copy_(torch.sort(torch.rand(rows, n, generator=g), 1)[1])
        b["count"].copy_(torch.randint(0, n + 1, (rows,), generator=g))

    fill(0)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            call()
    for seed in (1, 2, 3, 1):
        fill(seed)
        before = [p.clone() for p in kv.pools]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (out, token, lp, *kv.pools)]
        for p, x in zip(kv.pools, before):
            p.copy_(x)
        for x in (out, token, lp):
            x.fill_(7)
        call()
        torch.cuda.synchronize()
        for x, y in zip(got, (out, token, lp, *kv.pools)):
            assert torch.equal(x, y)


def test_calls_on_two_streams_at_once(dev):
    """Attention in parts (a workspace each), writing, drawing: two streams that wait for nothing of each other."""
    g = torch.Generator(device=dev).manual_seed(3)
    pages, rows = 200, 2
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).int().view(rows, -1).to(dev)
    kv_len = i32([1500, 900])
    mask = torch.ones(rows, 1, dtype=torch.int64, device=dev)
    inputs = []
    for _ in range(2):
        pool = torch.randint(0, 256, (pages, 2, H, 1040), generator=g, dtype=torch.uint8, device=dev)
        pool[..., 1024:] = 120
        x = torch.randn(3, rows, 1, H, 64, generator=g, device=dev).bfloat16()
        logits = torch.randn(rows, 5000, generator=g, device=dev)
        inputs.append((pool, x, logits, torch.rand(rows, generator=g, device=dev)))

    def step(pool, x, logits, u):
        q, k, v = x
        out = torch.empty_like(q)
        kernels.kv8_write(k[:, 0], v[:, 0], pool, table, kv_len - 1)
        kernels.attn_tree(q, pool, table, kv_len, mask, out, SCALE)
        return out, scoring.sample_tokens(logits, u, temperature=0.8, top_p=0.9).token

    want = [step(*a) for a in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(step(*inputs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for out, token in got[i]:
            assert torch.equal(out, want[i][0]) and torch.equal(token, want[i][1])
