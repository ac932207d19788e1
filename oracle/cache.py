"""Page state of a cache whose sequences share pages, one page at a time (plain
Python lists and a NumPy pool): what ``pts_cache_fork``, ``pts_cache_extend``,
``pts_cache_truncate`` and ``pts_cache_compact`` compute.

A page's count is the number of table entries that hold it; fresh pages are the
lowest free ones, as ``KvCachePool.allocate`` hands them out
(``flashinfer/cache_manager.py:89-97``); a shared partial page is copied before a
holder grows, as ``_copy_block`` does (``beam_search.py:92-96, 479-500``).
"""
from __future__ import annotations

from typing import List, Optional, Sequence

import numpy as np

BAD_INDEX, TWICE, TOO_LONG, NO_PAGES = 1, 2, 4, 8


def pages_of(tokens: int, page_len: int) -> int:
    return -(-tokens // page_len)


class PageState:
    """``pool`` [L, P, 2, page_len, H, D] or None (no bytes are moved)."""

    def __init__(self, rows: int, width: int, pages: int, page_len: int, pool: Optional[np.ndarray] = None):
        self.page_len, self.width = page_len, width
        self.refs = [0] * pages
        self.table = [[-1] * width for _ in range(rows)]
        self.lens = [0] * rows
        self.pool = pool

    def _pages(self, r: int) -> List[int]:
        return self.table[r][:pages_of(self.lens[r], self.page_len)]

    def fork(self, src: Sequence[int], dst: Sequence[int]) -> int:
        code = 0
        if any(not 0 <= r < len(self.table) for r in list(src) + list(dst)):
            code |= BAD_INDEX
        inside = [r for a, r in zip(src, dst) if 0 <= r < len(self.table) and 0 <= a < len(self.table)]
        if len(set(inside)) < len(inside):
            code |= TWICE
        if code:
            return code
        old = [(list(self.table[r]), self.lens[r]) for r in src]
        for r, (pages, n) in zip(dst, old):
            for p in self.table[r]:
                if p >= 0:
                    self.refs[p] -= 1
            for p in pages:
                if p >= 0:
                    self.refs[p] += 1
            self.table[r], self.lens[r] = list(pages), n
        return 0

    def extend(self, rows: Sequence[int], add: Sequence[int], groups: Optional[Sequence[int]] = None):
        """(status, page lists, lengths, shared leading pages per group); a call that cannot
        be done changes nothing and returns a batch of empty sequences."""
        code, seen, grow = 0, set(), []
        for r, a in zip(rows, add):
            if not 0 <= r < len(self.table) or a < 0:
                code |= BAD_INDEX
                continue
            if r in seen:
                code |= TWICE
            seen.add(r)
            if self.lens[r] + a > self.width * self.page_len:
                code |= TOO_LONG
        old = [self.lens[r] if 0 <= r < len(self.table) and a >= 0 else 0 for r, a in zip(rows, add)]
        if not code:
            tail = {}
            for i, (r, a) in enumerate(zip(rows, add)):
                if a > 0 and old[i] % self.page_len:
                    tail.setdefault(self.table[r][old[i] // self.page_len], []).append(i)
            need = []
            for i, (r, a) in enumerate(zip(rows, add)):
                first = pages_of(old[i], self.page_len)
                at = list(range(first, pages_of(old[i] + a, self.page_len)))
                if a > 0 and old[i] % self.page_len:
                    p = self.table[r][first - 1]
                    if self.refs[p] > 1 and not (len(tail[p]) == self.refs[p] and tail[p][-1] == i):
                        at.insert(0, first - 1)
                need += [(r, j, old[i]) for j in at]
            free = [p for p, n in enumerate(self.refs) if n == 0]
            if len(need) > len(free):
                code = NO_PAGES
        if not code:
            for (r, j, n), p in zip(need, free):
                q = self.table[r][j]
                if q >= 0:
                    self.refs[q] -= 1
                    if self.pool is not None:
                        k = n % self.page_len
                        self.pool[:, p, :, :k] = self.pool[:, q, :, :k]
                self.table[r][j] = p
                self.refs[p] = 1
            for r, a in zip(rows, add):
                self.lens[r] += a
        lists = [[] if code else self._pages(r) for r in rows]
        lens = [0 if code else self.lens[r] for r in rows]
        shared = []
        if groups is not None:
            for a, z in zip(groups[:-1], groups[1:]):
                n = 0
                while not code and a < z and all(n < old[i] // self.page_len and lists[i][n] == lists[a][n] for i in range(a, z)):
                    n += 1
                shared.append(n)
        return code, lists, lens, shared

    def truncate(self, rows: Sequence[int], new: Optional[Sequence[int]] = None) -> int:
        code = 0
        for i, r in enumerate(rows):
            if not 0 <= r < len(self.table):
                code = BAD_INDEX
                continue
            keep = min(self.lens[r], max(0, new[i]) if new is not None else 0)
            for j in range(pages_of(keep, self.page_len), pages_of(self.lens[r], self.page_len)):
                self.refs[self.table[r][j]] -= 1
                self.table[r][j] = -1
            self.lens[r] = keep
        return code

    def compact(self):
        """(refs, table, map, [live, moved]); moves the pool's pages."""
        live = [p for p, n in enumerate(self.refs) if n > 0]
        n = len(live)
        holes = iter([p for p in range(n) if self.refs[p] == 0])
        to = {p: p if p < n else next(holes) for p in live}
        refs = [0] * len(self.refs)
        for p in live:
            refs[to[p]] = self.refs[p]
            if self.pool is not None and to[p] != p:
                self.pool[:, to[p]] = self.pool[:, p]
        table = [[to.get(p, -1) for p in row] for row in self.table]
        return refs, table, [to.get(p, -1) for p in range(len(refs))], [n, sum(a != b for a, b in to.items())]
