"""Inputs and tolerances of the tree-attention tests (plain module, no tests)."""

import numpy as np
import torch

from oracle import kv8 as OK
from oracle import tree as OT

NAN = float("nan")


def tolerance(o, a):
    """Bound of |kernel - exact| per output.  The weights (of an 8-bit cache times V's power-of-two scales, which
    rounds nothing) are rounded to bf16 for the product with V: at most half a step, 2^-8 relative, each, so 2^-8 * a with a =
    sum_j w_j |v_j|; scores, exponentials and sums are fp32 (64-term products of values up to ~10, scores up to
    ~10: relative weight error < 1e-4); the result is rounded to bf16 once: 2^-8 |o|."""
    half = torch.finfo(torch.bfloat16).eps / 2
    e = (half + 1e-4) * a
    return e + half * (o.abs() + e) + 1e-30


def random_masks(rng, n, kind="tree"):
    """Masks of a row of n nodes, as Python integers."""
    if kind == "chain":
        return [2 ** (i + 1) - 1 for i in range(n)]
    if kind == "siblings":
        return [1 << i for i in range(n)]
    if kind == "full":  # a block: every node sees every node, bits past the row set as well
        return [2 ** 64 - 1] * n
    if kind == "none":
        return [0] * n
    masks = []
    for i in range(n):
        p = int(rng.integers(-1, i)) if i else -1
        masks.append(((masks[p] if p >= 0 else 0) | 1 << i) & 2 ** 64 - 1)  # a mask has 64 bits
    if kind == "padded":  # the last third stands for nothing
        for i in range(n - n // 3, n):
            masks[i] = 0
    return masks


class Case:
    """Rows of a paged cache whose pages and slots that no node sees hold NaN (8-bit: codes of an infinite scale), and
    whose table entries of pages that no node sees are out of range."""

    def __init__(self, *, n_nodes, kv_lens, H, bits, window=None, sinks=0, kind="tree", seed=0, packed=False, tail_q=0,
                 max_q=None, extra_cols=1):
        g = torch.Generator().manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.kv_lens, self.H, self.bits, self.packed = list(kv_lens), H, bits, packed
        self.window, self.sinks, self.max_q = window, sinks, max_q
        rows = len(kv_lens)
        cols = max(1, max((x + 15) // 16 for x in kv_lens)) + extra_cols
        n_pages = sum((x + 15) // 16 for x in kv_lens) + 3
        order = rng.permutation(n_pages)
        table = rng.choice([-5, n_pages, 2**31 - 1, -2**31], size=(rows, cols)).astype(np.int64)
        if bits == 16:
            pool = torch.full((n_pages, 2, H, 1024), NAN, dtype=torch.bfloat16)
        else:
            pool = torch.randint(-128, 128, (n_pages, 2, H, 1040), generator=g, dtype=torch.int8).view(torch.uint8)
            pool[..., 1024:] = 255
        self.n_q = sum(n_nodes) + tail_q
        self.q = (2 * torch.randn(self.n_q, H, 64, generator=g)).bfloat16()
        self.starts = [int(x) for x in np.concatenate([[0], np.cumsum(n_nodes)])]
        self.ref = torch.full((self.n_q, H, 64), 77.0, dtype=torch.float64)
        self.tol = torch.zeros(self.n_q, H, 64, dtype=torch.float64)
        all_masks = []
        at = 0
        for r, (n, kv) in enumerate(zip(n_nodes, kv_lens)):
            masks = random_masks(rng, n, kind)
            all_masks += masks
            npg = (kv + 15) // 16
            kvs = 1.0 * torch.randn(2, npg * 16, H, 64, generator=g)
            # some tokens much larger or smaller in V, so that scales differ
            kvs[1] *= torch.pow(2.0, torch.randint(-3, 4, (npg * 16, H, 1), generator=g))
            kvs = kvs.bfloat16()
            top = n if max_q is None else min(n, max_q)
            see = OT.visible(kv, n, masks[:top], window, sinks)
            some = torch.cat([see.any(0), torch.zeros(npg * 16 - kv, dtype=torch.bool)])
            pages = order[at:at + npg]
            at += npg
            used = some.view(npg, 16).any(1).numpy()
            table[r, :npg][used] = pages[used]
            if bits == 8:
                codes, scales = OK.quantise(kvs)
                exact = OK.values(codes, scales)
                scales[:, ~some] = 255
                for j in range(npg * 16):
                    for plane in (0, 1):
                        OK.write(pool, int(pages[j // 16]), j % 16, plane, codes[plane, j], scales[plane, j])
            else:
                exact = kvs.double()
                kvs[:, ~some] = NAN
                pg = torch.from_numpy(pages)
                pool[pg, 0] = kvs[0].view(npg, 16, H, 64).permute(0, 2, 1, 3).reshape(npg, H, 1024)
                pool[pg, 1] = kvs[1].view(npg, 16, H, 64).permute(0, 2, 3, 1).reshape(npg, H, 1024)
            s = slice(self.starts[r], self.starts[r] + top)
            o, a = OT.attend(self.q[s], exact[0, :kv], exact[1, :kv], see, 0.125)
            self.ref[s], self.tol[s] = o, tolerance(o, a)
        all_masks += [1] * tail_q
        self.mask = torch.from_numpy(np.array(all_masks, dtype=np.uint64).view(np.int64))
        self.pool, self.table = pool, torch.from_numpy(table.astype(np.int32))

    def device(self, dev):
        d = lambda x: x.to(dev)  # noqa: E731
        rows = len(self.kv_lens)
        shape = (self.n_q,) if self.packed else (rows, self.n_q // rows)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
        return dict(q=d(self.q).view(*shape, self.H, 64), mask=d(self.mask).view(shape), pool=d(self.pool),
                    table=d(self.table), kv_len=i32(self.kv_lens), q_start=i32(self.starts) if self.packed else None)

    def run(self, dev, kernels, **kw):
        t = self.device(dev)
        out = torch.full_like(t["q"], 77.0)
        if self.max_q is not None:
            kw.setdefault("max_q", self.max_q)
        kernels.attn_tree(t["q"], t["pool"], t["table"], t["kv_len"], t["mask"], out, 0.125, window=self.window,
                          sinks=self.sinks, q_start=t["q_start"], **kw)
        torch.cuda.synchronize()
        return out

    def check(self, out):
        """Rows that are not computed hold the 77 that they came with."""
        out = out.cpu().double().view(self.n_q, self.H, 64)
        err = (out - self.ref).abs()
        bad = ~(err <= self.tol)  # NaN fails too
        assert not bool(bad.any()), (f"{int(bad.sum())} of {bad.numel()} values off, first at {bad.nonzero()[0].tolist()}, "
                                     f"worst {err.nan_to_num(1e9).max().item():.4g}")
