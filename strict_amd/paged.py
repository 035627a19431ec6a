"""A KV cache in pages for a batch of sequences: the host's bookkeeping
(`PageTable`) and the cache on the device that follows it (`PagedCache`), which
`Context.qk_norm_rope_paged` fills and `Context.attn_paged` reads.

Sequences share pages after a fork; a page that more than one sequence holds is
copied when one of them appends to it. The reference has no counterpart.
"""
from __future__ import annotations

import heapq
import operator

import numpy as np

from . import Context, PagedKV, PagedKV8


class OutOfPages(RuntimeError):
    """A sequence needs more pages than the pool (or its table) has."""


class PageTable:
    """Which pages each row's sequence holds. Copies that its methods return,
    (from, to) pairs, are due before the pages are written; nothing changes
    when a method raises."""

    def __init__(self, rows: int, max_pages: int, num_pages: int, page_size: int):
        if min(rows, max_pages, num_pages, page_size) < 1:
            raise ValueError("rows, max_pages, num_pages and page_size must be positive")
        self.max_pages, self.num_pages, self.page_size = max_pages, num_pages, page_size
        self.pages = [[] for _ in range(rows)]
        self.lengths = [0] * rows
        self.holders = [0] * num_pages
        self._free = list(range(num_pages))  # a heap: the lowest number first

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _check(self, row: int) -> None:
        if not 0 <= row < len(self.pages):
            raise IndexError(f"row {row} of {len(self.pages)}")

    def extend(self, new) -> list:
        """Room for new[row] more tokens in every row named in the mapping, all or none."""
        plan, need = [], 0
        for row, n in new.items():
            self._check(row)
            n = operator.index(n)
            if n < 0:
                raise ValueError("a negative number of tokens")
            pages, length = self.pages[row], self.lengths[row]
            total = -(-(length + n) // self.page_size)
            if total > self.max_pages:
                raise OutOfPages(f"row {row}: {total} pages, its table holds {self.max_pages}")
            # the last page, if tokens of a shared one would be followed by this row's own
            split = n > 0 and length % self.page_size != 0 and self.holders[pages[-1]] > 1
            plan.append((row, n, total - len(pages), split))
            need += total - len(pages)
        # a page shared by these rows alone stays with the last of them
        held = {}
        for row, _, _, split in plan:
            if split:
                held[self.pages[row][-1]] = held.get(self.pages[row][-1], 0) + 1
        need += sum(n - (self.holders[page] == n) for page, n in held.items())
        if need > len(self._free):
            raise OutOfPages(f"{need} pages needed, {len(self._free)} free")
        copies = []
        for row, n, more, split in plan:
            pages = self.pages[row]
            if split and self.holders[pages[-1]] > 1:
                old, page = pages[-1], heapq.heappop(self._free)
                copies.append((old, page))
                self.holders[old] -= 1
                self.holders[page] = 1
                pages[-1] = page
            for _ in range(more):
                page = heapq.heappop(self._free)
                self.holders[page] = 1
                pages.append(page)
            self.lengths[row] += n
        return copies

    def fork(self, row: int, to: int) -> None:
        """Row `to`, which must be empty, continues from the same tokens as `row`."""
        self._check(row)
        self._check(to)
        if self.pages[to] or self.lengths[to]:
            raise ValueError(f"row {to} is not empty")
        self.pages[to] = list(self.pages[row])
        self.lengths[to] = self.lengths[row]
        for page in self.pages[to]:
            self.holders[page] += 1

    def free(self, row: int) -> None:
        """Ends row's sequence; pages that no other row holds are free again."""
        self._check(row)
        for page in self.pages[row]:
            self.holders[page] -= 1
            if self.holders[page] == 0:
                heapq.heappush(self._free, page)
        self.pages[row] = []
        self.lengths[row] = 0

    def compact(self) -> list:
        """Moves the pages in use to the lowest numbers."""
        used = self.num_pages - len(self._free)
        to = sorted(p for p in self._free if p < used)
        moved = [p for p in range(used, self.num_pages) if self.holders[p]]
        at = dict(zip(moved, to))
        for old, new in at.items():
            self.holders[new], self.holders[old] = self.holders[old], 0
        self.pages = [[at.get(p, p) for p in pages] for pages in self.pages]
        self._free = list(range(used, self.num_pages))
        return list(at.items())

    def array(self) -> np.ndarray:
        """The table as the kernels read it: int32 [rows, max_pages], -1: no page."""
        t = np.full((len(self.pages), self.max_pages), -1, np.int32)
        for row, pages in enumerate(self.pages):
            t[row, :len(pages)] = pages
        return t


class PagedCache:
    """K and V of `layers` layers in pages on a context's device, for up to `rows`
    sequences of up to max_pages pages each: as 16-bit values of `dtype`, or with bits=8
    quantised as they are written (E4M3 with a power of two for each row), `dtype` being
    that of the activations. Every method is ordered on the
    context's stream; `step`, and `compact` where it moves pages, upload tables from
    the host and wait for the stream, and are not to be captured."""

    def __init__(self, ctx: Context, layers: int, kv_heads: int, head_dim: int, *, rows: int,
                 max_pages: int, num_pages: int, page_size: int = 64, dtype: str = "f16", bits: int = 16):
        if bits not in (8, 16):
            raise ValueError(f"{bits} bits: 8 or 16")
        self.ctx, self.layers = ctx, layers
        self.table = PageTable(rows, max_pages, num_pages, page_size)
        if bits == 16:
            self.page_bytes = kv_heads * page_size * head_dim * 2
            self.planes = 2 * layers  # [layer][k, v][page]
        else:
            self.page_bytes = PagedKV8.page_bytes(kv_heads, page_size, head_dim)
            self.planes = layers  # [layer][page]
        plane = num_pages * self.page_bytes
        self.buffers = []
        try:
            self.pool = self._keep(ctx.alloc(self.planes * plane))
            self.table_buf = self._keep(ctx.empty((rows, max_pages), np.int32))
            self.lengths = self._keep(ctx.empty(rows, np.int32))
            self.starts = self._keep(ctx.empty(rows + 1, np.int32))
            self.moves = self._keep(ctx.empty((2, num_pages), np.int32))
            kind, planes = (PagedKV, 2) if bits == 16 else (PagedKV8, 1)
            self.kv = [kind(*(self.pool.ptr + (planes * i + j) * plane for j in range(planes)),
                            self.table_buf, self.lengths, self.starts, batch=rows,
                            max_pages=max_pages, num_pages=num_pages, page_size=page_size,
                            kv_heads=kv_heads, head_dim=head_dim, dtype=dtype)
                       for i in range(layers)]  # a layer's view, for the operators
            self._upload({})
        except BaseException:
            self.dispose()
            raise

    def _keep(self, buffer):
        self.buffers.append(buffer)
        return buffer

    def _copy(self, pairs) -> None:
        if pairs:
            src, dst = (np.array(p, np.int32) for p in zip(*pairs))
            num = self.table.num_pages
            at_src, at_dst = self.moves.view(0, 4 * num), self.moves.view(4 * num, 4 * num)
            at_src.copy_from_host(src)
            at_dst.copy_from_host(dst)
            self.ctx.pages_copy(self.pool, self.planes, num, self.page_bytes, at_src, at_dst,
                                len(pairs))

    def _upload(self, new) -> None:
        rows = len(self.table.lengths)
        starts = np.concatenate([[0], np.cumsum([new.get(r, 0) for r in range(rows)])])
        self.table_buf.copy_from_host(self.table.array())
        self.lengths.copy_from_host(np.array(self.table.lengths, np.int32))
        self.starts.copy_from_host(starts.astype(np.int32))

    def step(self, new) -> int:
        """Prepares a step of new[row] new tokens for the rows named (their rows in
        the step's tensors follow the rows' order); returns how many there are."""
        new = {row: operator.index(n) for row, n in dict(new).items()}
        self._copy(self.table.extend(new))
        self._upload(new)
        return sum(new.values())

    def fork(self, row: int, to: int) -> None:
        self.table.fork(row, to)

    def free(self, row: int) -> None:
        self.table.free(row)

    def compact(self) -> int:
        """Moves the pages in use to the lowest numbers; returns how many moved. The
        operators see the new places from the next step on."""
        moves = self.table.compact()
        self._copy(moves)
        return len(moves)

    def dispose(self) -> None:
        for b in self.buffers:
            b.free()

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.dispose()
