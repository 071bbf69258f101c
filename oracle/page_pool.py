"""Page bookkeeping and page contents of a paged cache, one page at a time.

``Pool`` mirrors the device state of the page operations: reference counts,
row page lists, and the contents of every layer.  A new page is always the
lowest free id; requests are served in row order, all or nothing.
"""

from __future__ import annotations

import copy

import numpy as np


class Refused(Exception):
    pass


class Pool:
    def __init__(self, data: np.ndarray, refcount, rows: list[list[int]], last: list[int], cap: int) -> None:
        self.data = data  # [layers, pages, 2, page_size, ...]
        self.ps = data.shape[3]
        self.refcount = list(refcount)
        self.rows = [list(r) for r in rows]
        self.last = list(last)
        self.cap = cap

    def length(self, r: int) -> int:
        return (len(self.rows[r]) - 1) * self.ps + self.last[r] if self.rows[r] else 0

    def _take(self) -> int:
        for p, c in enumerate(self.refcount):
            if c == 0:
                self.refcount[p] = 1
                return p
        raise Refused("exhausted")

    def _atomic(self, fn) -> None:
        saved = copy.deepcopy((self.refcount, self.rows, self.last)), self.data.copy()
        try:
            fn()
        except Refused:
            (self.refcount, self.rows, self.last), self.data[...] = saved
            raise

    def release(self, rows) -> None:
        for r in rows:
            for p in self.rows[r]:
                self.refcount[p] -= 1
            self.rows[r], self.last[r] = [], 0

    def reserve(self, counts) -> list[tuple[int, int]]:
        slots: list[tuple[int, int]] = []

        def go() -> None:
            for r, n in enumerate(counts):
                length = self.length(r)
                if n and length % self.ps and self.refcount[self.rows[r][-1]] != 1:
                    raise Refused("shared")
                if -(-(length + n) // self.ps) > self.cap:
                    raise Refused("capacity")
            for r, n in enumerate(counts):
                for _ in range(n):
                    if self.length(r) % self.ps == 0:
                        self.rows[r].append(self._take())
                        self.last[r] = 0
                    slots.append((self.rows[r][-1], self.last[r]))
                    self.last[r] += 1

        self._atomic(go)
        return slots

    def fork(self, src, dst) -> None:
        def go() -> None:
            inside = all(0 <= r < len(self.rows) for r in [*src, *dst])
            if not inside or len(set(dst)) != len(dst) or set(src) & set(dst) or any(self.rows[d] for d in dst):
                raise Refused("rows")
            for s, d in zip(src, dst):
                row = list(self.rows[s])
                if row and self.last[s] < self.ps:
                    p = self._take()
                    self.data[:, p, :, : self.last[s]] = self.data[:, row[-1], :, : self.last[s]]
                    row[-1] = p
                    shared = row[:-1]
                else:
                    shared = row
                for p in shared:
                    self.refcount[p] += 1
                self.rows[d], self.last[d] = row, self.last[s]

        self._atomic(go)

    def compact(self, keep_from, keep) -> None:
        def go() -> None:
            counts = list(self.refcount)  # decisions are made on the state before the call
            old_rows = [list(r) for r in self.rows]
            for r, (kf, kept) in enumerate(zip(keep_from, keep)):
                order = list(range(kf)) + list(kept)
                if len(order) > self.length(r):
                    raise Refused("length")
                stays = 0
                while stays < len(order) and order[stays] == stays:
                    stays += 1
                full = stays // self.ps
                rest = len(order) - full * self.ps
                if stays == len(order) and (rest == 0 or counts[old_rows[r][full]] == 1):
                    self.rows[r] = old_rows[r][: full + (rest > 0)]
                else:
                    new = [self._take() for _ in range(-(-rest // self.ps))]
                    for i in range(full * self.ps, len(order)):
                        a, b = old_rows[r][order[i] // self.ps], new[i // self.ps - full]
                        self.data[:, b, :, i % self.ps] = self.data[:, a, :, order[i] % self.ps]
                    self.rows[r] = old_rows[r][:full] + new
                self.last[r] = (len(order) - 1) % self.ps + 1 if order else 0
            for r, row in enumerate(old_rows):
                for p in row:
                    if p not in self.rows[r]:
                        self.refcount[p] -= 1

        self._atomic(go)
