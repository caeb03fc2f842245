"""Paged KV pool, page tables and the attention plan (host side of kernel (a)).

The reference gives each sample a static slice of ``ceil(max_seq/16)`` pages
(engines/flashinfer.py:104-116) and re-plans the attention metadata in Python
per block (engines/flashinfer.py:346-411, 1506-1556).  Here every layer owns a
zero-filled pool ``[pages, 2, H, 16*64]`` (layout in csrc/kv_layout.h), rows
map positions to pages through an int32 table that may be any permutation of
pool pages, and the attention work list is built once per block by the
native planner (``yapd_attn_plan``) and uploaded.

:class:`SharedPagedKV` maps pages on demand instead of a slice per row: rows
share a prefix by reference count, pages behind an attention window go back to
the pool, and the pool is compacted.
"""

from __future__ import annotations

from typing import List, Optional, Sequence

import numpy as np
import torch

from . import kernels

PAGE_SIZE = 16
HEAD_DIM = 64


def to_device_async(data, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """Host data (list or array) on ``device`` without a host synchronisation: staged through
    pinned memory and copied on the current stream (a copy from pageable memory would wait for
    every kernel already queued)."""
    t = torch.as_tensor(np.asarray(data), dtype=dtype)
    if torch.device(device).type != "cuda":
        return t.to(device)
    return t.pin_memory().to(device, non_blocking=True)


def copy_from_host_async(dst: torch.Tensor, data) -> None:
    """``dst.copy_(data)`` for host data (list or array) without a host synchronisation: staged
    through pinned memory and copied on the current stream.  Not for use inside a graph capture
    (the copy would keep reading a recycled staging buffer on every replay)."""
    t = torch.as_tensor(np.asarray(data)).to(dst.dtype)
    if dst.device.type != "cuda":
        dst.copy_(t)
        return
    dst.copy_(t.pin_memory(), non_blocking=True)


def _check_bits(kv_bits: int) -> int:
    kernels.require(kv_bits in (8, 16), f"kv_bits must be 8 or 16, got {kv_bits}")
    return int(kv_bits)


class PagedKV:
    """Per-layer page pools plus a host-side page allocator and device page table."""

    def __init__(self, *, n_layers: int, n_rows: int, pages_per_row: int, n_heads: int,
                 device: torch.device, n_pages: Optional[int] = None, shuffle_seed: Optional[int] = None,
                 kv_bits: int = 16):
        """``kv_bits`` 8: uint8 pools of codes and scales (``kernels.kv8_write``), half the bytes; 16: bf16."""
        self.kv_bits = _check_bits(kv_bits)
        self.n_layers = int(n_layers)
        self.n_rows = int(n_rows)
        self.pages_per_row = int(pages_per_row)
        self.n_heads = int(n_heads)
        self.device = torch.device(device)
        self.n_pages = int(n_pages) if n_pages is not None else self.n_rows * self.pages_per_row
        kernels.require(self.n_pages >= self.n_rows * self.pages_per_row, "pool smaller than rows * pages_per_row")
        self._make_pools()
        order = np.arange(self.n_pages, dtype=np.int32)
        if shuffle_seed is not None:
            order = np.random.default_rng(shuffle_seed).permutation(self.n_pages).astype(np.int32)
        take = order[: self.n_rows * self.pages_per_row]
        self.table_host = take.reshape(self.n_rows, self.pages_per_row).copy()
        self.table = torch.from_numpy(self.table_host).to(self.device)

    def _make_pools(self) -> None:
        tile, dtype = (kernels.TILE8, torch.uint8) if self.kv_bits == 8 else (PAGE_SIZE * HEAD_DIM, torch.bfloat16)
        self.pools: List[torch.Tensor] = [
            torch.zeros(self.n_pages, 2, self.n_heads, tile, dtype=dtype, device=self.device)
            for _ in range(self.n_layers)
        ]

    @property
    def bytes_per_layer(self) -> int:
        return self.pools[0].numel() * self.pools[0].element_size()

    def swap_rows(self, a: int, b: int) -> None:
        """Exchange page-table rows ``a`` and ``b`` (host mirror and device table): each row's KV
        moves with its pages, nothing is copied.  Device work is stream-ordered, no host sync."""
        if a == b:
            return
        self.table_host[[a, b]] = self.table_host[[b, a]]
        tmp = self.table[a].clone()
        self.table[a].copy_(self.table[b])
        self.table[b].copy_(tmp)

    def copy_pages(self, src, dst) -> None:
        """``pool[dst[i]] = pool[src[i]]`` in every layer's pool for host page ids (see
        :func:`kernels.kv_copy_pages`), on the current stream; torch's index operations, with the same
        refusals, on the CPU."""
        if self.device.type == "cuda":
            kernels.kv_copy_pages(self.pools, src, dst)
            return
        src, dst = kernels.page_ids(src, "src"), kernels.page_ids(dst, "dst")
        for pool in self.pools:
            kernels.check_page_pairs(src, dst, pool.shape[0])
        src_t, dst_t = (torch.from_numpy(x.astype(np.int64)) for x in (src, dst))
        for pool in self.pools:
            pool.index_copy_(0, dst_t, pool.index_select(0, src_t))

    def keep_nodes(self, base: torch.Tensor, kept: torch.Tensor, n_kept: torch.Tensor) -> None:
        """Move the accepted nodes of every row's drafted tree to the positions from ``base`` on, in every layer (see
        :func:`kernels.kv_keep`; entry ``r`` of the device tensors is the cache's row ``r``), on the current stream.  A
        :class:`SharedPagedKV` must have all of a tree's positions reserved: an unmapped one is page 0's, whose
        bytes would be kept as the node's."""
        kernels.kv_keep(self.pools, self.table, base, kept, n_kept)

    def copy_row_pages(self, src_row: int, dst_row: int, n_positions: int) -> None:
        """Copy the pages holding positions ``[0, n_positions)`` of one row to another, every layer."""
        npg = (n_positions + PAGE_SIZE - 1) // PAGE_SIZE
        src, dst = self.table_host[src_row, :npg].copy(), self.table_host[dst_row, :npg].copy()
        targets = set(dst.tolist())
        if len(targets) == len(dst) and targets.isdisjoint(src.tolist()):
            self.copy_pages(src, dst)
            return
        # rows that share pages: every source is read before any page is written
        src_t, dst_t = (to_device_async(x, torch.int64, self.device) for x in (src, dst))
        for pool in self.pools:
            pool.index_copy_(0, dst_t, pool.index_select(0, src_t))


class SharedPagedKV(PagedKV):
    """A paged KV cache whose rows map pages on demand and share them by reference count.

    A row maps a page when :meth:`reserve` first covers one of its positions; :meth:`fork` gives other
    rows the same pages (the partial last one as a copy of their own); :meth:`release` and
    :meth:`release_before` give pages back; :meth:`compact` moves the mapped pages to the pool's front.
    Table entries that map nothing name page 0, which is never handed out: it takes stray writes and
    holds nothing.  Attention must not see positions whose page was released (``kernels.attn_window``
    does not, for a window no longer than what was kept).

    The bookkeeping is on the host and takes effect at once; table uploads and page copies go to the
    current stream, which has to be the one (or ordered with the one) that the cache is used on.  Not
    for use inside a graph capture; a captured launch reads the tables and pools, whose addresses stay.
    """

    def __init__(self, *, n_layers: int, n_rows: int, pages_per_row: int, n_heads: int, device: torch.device,
                 n_pages: int, kv_bits: int = 16):
        """``n_pages`` counts the pool's pages, page 0 included; a row maps at most ``pages_per_row``; ``kv_bits`` as
        :class:`PagedKV` has it."""
        self.kv_bits = _check_bits(kv_bits)
        kernels.require(n_layers >= 1 and n_rows >= 1 and pages_per_row >= 1 and n_heads >= 1 and n_pages >= 2,
                        "need at least one layer, row, page per row and head, and two pages")
        self.n_layers = int(n_layers)
        self.n_rows = int(n_rows)
        self.pages_per_row = int(pages_per_row)
        self.n_heads = int(n_heads)
        self.device = torch.device(device)
        self.n_pages = int(n_pages)
        self._make_pools()
        self.table_host = np.zeros((self.n_rows, self.pages_per_row), dtype=np.int32)
        self.table = torch.zeros(self.n_rows, self.pages_per_row, dtype=torch.int32, device=self.device)
        self._refs = np.zeros(self.n_pages, dtype=np.int32)
        self._refs[0] = 1
        self._free = list(range(self.n_pages - 1, 0, -1))  # the lowest free page is handed out first

    @property
    def free_pages(self) -> int:
        """Pages that :meth:`reserve` and :meth:`fork` can still take."""
        return len(self._free)

    def refcount(self, page: int) -> int:
        """Rows that map ``page``."""
        return int(self._refs[page])

    # ------------------------------------------------------------------ #

    def _check_row(self, row: int) -> None:
        kernels.require(0 <= row < self.n_rows, f"row {row} outside [0, {self.n_rows})")

    def _check_free(self, n: int, given_back: int = 0) -> None:
        free = len(self._free) + given_back
        if n > free:
            raise RuntimeError(f"the pool is out of pages: {n} needed, {free} free")

    def _take(self, n: int) -> List[int]:
        self._check_free(n)
        return [self._free.pop() for _ in range(n)]

    def _drop(self, pages: np.ndarray) -> None:
        """One reference of each page (ids of mapped entries, repeats allowed) is gone."""
        np.subtract.at(self._refs, pages, 1)
        gone = np.unique(pages)
        self._free.extend(gone[self._refs[gone] == 0][::-1].tolist())

    def _upload(self, rows: Sequence[int]) -> None:
        a, b = min(rows), max(rows) + 1
        copy_from_host_async(self.table[a:b], self.table_host[a:b].copy())

    def reserve(self, row: int, begin: int, end: int) -> None:
        """Map positions ``[begin, end)`` of ``row`` to pages that no other row shares, so that they can be
        written: an unmapped page is taken from the pool, a shared one replaced by a copy.  Raises
        ``RuntimeError``, with nothing changed, if the pool has too few pages left."""
        self._check_row(row)
        kernels.require(0 <= begin <= end <= self.pages_per_row * PAGE_SIZE,
                        f"positions [{begin}, {end}) outside what a row maps")
        if begin == end:
            return
        c0, c1 = begin // PAGE_SIZE, (end - 1) // PAGE_SIZE + 1
        now = self.table_host[row, c0:c1]
        new = np.nonzero((now == 0) | (self._refs[now] > 1))[0]
        if not len(new):
            return
        old, pages = now[new].copy(), np.asarray(self._take(len(new)), dtype=np.int32)
        self.table_host[row, c0 + new] = pages
        self._refs[pages] = 1
        shared = old != 0
        if shared.any():
            self.copy_pages(old[shared], pages[shared])
            self._drop(old[shared])
        self._upload([row])

    def fork(self, src_row: int, dst_rows: Sequence[int], n_positions: int) -> None:
        """Give every row of ``dst_rows`` (rows that map nothing) the first ``n_positions`` positions of
        ``src_row``: whole pages are shared, a partial last page is copied, one copy a row, all in one
        launch.  What of the source was released stays unmapped."""
        rows = [int(r) for r in dst_rows]
        for r in (src_row, *rows):
            self._check_row(r)
        kernels.require(len(set(rows)) == len(rows) and src_row not in rows, "a fork's rows must be distinct")
        kernels.require(0 <= n_positions <= self.pages_per_row * PAGE_SIZE, "n_positions outside what a row maps")
        kernels.require(not self.table_host[rows].any(), "a fork's destination rows must map nothing")
        if not rows or n_positions == 0:
            return
        whole, part = divmod(n_positions, PAGE_SIZE)
        tail = int(self.table_host[src_row, whole]) if part else 0
        own = self._take(len(rows)) if tail else []
        shared = self.table_host[src_row, :whole]
        self.table_host[rows, :whole] = shared
        self._refs[shared[shared != 0]] += len(rows)
        if tail:
            self.table_host[rows, whole] = own
            self._refs[own] = 1
            self.copy_pages([tail] * len(own), own)
        self._upload(rows)

    def release(self, row: int) -> None:
        """Unmap every page of ``row``."""
        self._release(row, np.arange(self.pages_per_row))

    def release_before(self, row: int, position: int, sinks: int = 0) -> None:
        """Unmap the pages of ``row`` whose positions all lie in ``[sinks, position)``: what a window that
        begins at ``position``, with ``sinks`` first tokens kept, no longer sees.  Nothing for a ``position``
        of 0 or less."""
        kernels.require(sinks >= 0, "sinks must be >= 0")
        first = (sinks + PAGE_SIZE - 1) // PAGE_SIZE
        self._release(row, np.arange(first, min(position // PAGE_SIZE, self.pages_per_row)))

    def _release(self, row: int, cols: np.ndarray) -> None:
        self._check_row(row)
        cols = cols[self.table_host[row, cols] != 0]
        if not len(cols):
            return
        self._drop(self.table_host[row, cols])
        self.table_host[row, cols] = 0
        self._upload([row])

    def compact(self) -> int:
        """Move the mapped pages to the pool's front (one launch, and an upload of the table); returns how
        many pages are in use, page 0 included: pages from there on hold nothing."""
        live = np.nonzero(self._refs)[0]
        n = len(live)
        src = live[live >= n]
        if len(src):
            dst = np.nonzero(self._refs[:n] == 0)[0]  # as many holes in front as pages behind
            self.copy_pages(src, dst)
            where = np.arange(self.n_pages, dtype=np.int32)
            where[src] = dst
            self.table_host = where[self.table_host]
            self._refs[dst] = self._refs[src]
            self._refs[src] = 0
            self._upload([0, self.n_rows - 1])
        self._free = list(range(self.n_pages - 1, n - 1, -1))
        return n

    def copy_row_pages(self, src_row: int, dst_row: int, n_positions: int) -> None:
        """Positions ``[0, n_positions)`` of ``src_row`` as pages of ``dst_row``'s own; what the destination
        mapped there is given back first.  Unmapped source pages stay unmapped.  Raises ``RuntimeError``,
        with nothing changed, if the pool has too few pages left."""
        self._check_row(src_row)
        self._check_row(dst_row)
        kernels.require(0 <= n_positions <= self.pages_per_row * PAGE_SIZE, "n_positions outside what a row maps")
        if src_row == dst_row or n_positions == 0:
            return
        cols = np.arange((n_positions + PAGE_SIZE - 1) // PAGE_SIZE)
        src = self.table_host[src_row, cols]
        mapped = src != 0
        old = self.table_host[dst_row, cols]
        old = old[old != 0]
        self._check_free(int(mapped.sum()), int((self._refs[old] == 1).sum()))
        self._drop(old)  # first, so that its own pages can be taken again; the source's are still mapped by it
        own = self._take(int(mapped.sum()))
        new = np.zeros_like(src)
        new[mapped] = own
        self._refs[own] = 1
        self.copy_pages(src[mapped], own)
        self.table_host[dst_row, cols] = new
        self._upload([dst_row])


class AttnPlan:
    """Device work list + split-KV workspace for one set of per-row kv lengths."""

    def __init__(self, kv_len: Sequence[int], bl: int, n_heads: int, device: torch.device,
                 target_items: int = 192, min_split_keys: int = 1024):
        work, merge, n_slots = kernels.attn_plan(kv_len, target_items=target_items, min_split_keys=min_split_keys)
        self.kv_len_host = [int(x) for x in kv_len]
        self._max_kv_len = max(self.kv_len_host)  # of the planned lengths, which do not change
        self.work = to_device_async(work, torch.int32, device)
        self.merge = to_device_async(merge, torch.int32, device) if merge.shape[0] else None
        self.n_slots = n_slots
        self.kv_len = to_device_async(self.kv_len_host, torch.int32, device)
        if n_slots:
            self.part_o = torch.empty(n_slots, bl, n_heads, HEAD_DIM, dtype=torch.float32, device=device)
            self.part_ml = torch.empty(n_slots, bl, n_heads, 2, dtype=torch.float32, device=device)
        else:
            self.part_o = self.part_ml = None

    def run(self, q: torch.Tensor, pool: torch.Tensor, table: torch.Tensor, out: torch.Tensor,
            scale: float, causal: bool = False) -> None:
        kernels.require(self._max_kv_len <= table.shape[1] * PAGE_SIZE,
                        "page table maps fewer positions than kv_len")
        kernels.attn_paged_block(q, pool, table, self.kv_len, self.work, self.merge, self.part_o, self.part_ml,
                                 out, scale, causal=causal)
