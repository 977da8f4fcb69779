"""The paged cache's definition in plain Python and 64 bits, for the tests of
verbo_b200/cache.py: tables and reference counts one entry after the other, codes
from the list of e4m3's values."""
from __future__ import annotations

import numpy as np

# the values of codes 0..126 in ascending order; 127 is NaN
GRID = np.array([(m / 8.0) * 2.0**-6 if e == 0 else (1 + m / 8.0) * 2.0**(e - 7) for e in range(16) for m in range(8)])[:127]


def decode(codes):
    codes = np.asarray(codes, dtype=np.uint8)
    mag = codes & 0x7F
    v = np.where(mag == 127, np.nan, GRID[np.minimum(mag, 126)])
    return np.where(codes & 0x80, -v, v)


def encode(x):
    """Nearest code, ties to even, saturating; NaN to NaN."""
    x = np.asarray(x, dtype=np.float64)
    mag = np.minimum(np.abs(np.where(np.isnan(x), 0, x)), 448.0)
    hi = np.minimum(np.searchsorted(GRID, mag), 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = mag - GRID[lo], GRID[hi] - mag
    c = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi).astype(np.uint8)
    c = np.where(np.signbit(x), c | 0x80, c).astype(np.uint8)
    return np.where(np.isnan(x), 0x7F, c)


def scale_for(x):
    """Smallest power of two s >= 2^-64 with |x| <= 448 s for the finite x."""
    x = np.abs(x[np.isfinite(x)])
    most = x.max() if x.size else 0.0
    q = -64
    while most > 448.0 * 2.0**q:
        q += 1
    return 2.0**q


class Model:
    def __init__(self, k, v, ks, vs, table, lens, refs):
        """numpy arrays (codes as uint8), copied"""
        self.k, self.v, self.ks, self.vs = k.copy(), v.copy(), ks.copy(), vs.copy()
        self.table, self.lens, self.refs = table.copy(), lens.copy(), refs.copy()
        self.page = k.shape[3]

    def used(self, n):
        return -(-int(n) // self.page)

    def reserve(self, add):
        rows, width = self.table.shape
        start = np.full(rows, -1, dtype=np.int32)
        for r in range(rows):
            if add[r] > 0 and int(self.lens[r]) + int(add[r]) > width * self.page:
                return start, -(r + 1)
        refs, table = self.refs.copy(), self.table.copy()
        free = [p for p in range(refs.size) if refs[p] == 0]
        copies, missing, taken = [], 0, 0

        def take():
            nonlocal missing, taken
            taken += 1
            if taken > len(free):
                missing += 1
                return -1
            refs[free[taken - 1]] = 1
            return free[taken - 1]

        for r in range(rows):
            n, a = int(self.lens[r]), int(add[r])
            if a <= 0:
                continue
            if n % self.page:
                p = table[r, n // self.page]
                if refs[p] > 1:
                    refs[p] -= 1
                    to = take()
                    copies.append((p, to))
                    table[r, n // self.page] = to
            for j in range(self.used(n), self.used(n + a)):
                table[r, j] = take()
        if missing:
            return start, missing
        for r in range(rows):
            if add[r] > 0:
                start[r] = self.lens[r]
                self.lens[r] += add[r]
        self.table, self.refs = table, refs
        for s, d in copies:
            self.move(s, d)
        return start, 0

    def move(self, s, d):
        for t in (self.k, self.v, self.ks, self.vs):
            t[:, d] = t[:, s]

    def fork(self, parents, beams):
        table, lens = self.table.copy(), self.lens.copy()
        for r in range(table.shape[0]):
            p = int(parents[r // beams, r % beams])
            for e in table[r, :self.used(lens[r])]:
                self.refs[e] -= 1
            if 0 <= p < beams:
                src = r // beams * beams + p
                self.table[r], self.lens[r] = table[src], lens[src]
            else:
                self.table[r], self.lens[r] = -1, 0
        for r in range(table.shape[0]):
            for e in self.table[r, :self.used(self.lens[r])]:
                self.refs[e] += 1

    def free(self, keep):
        for r in range(self.table.shape[0]):
            if 0 <= keep[r] < self.lens[r]:
                for j in range(self.used(keep[r]), self.used(self.lens[r])):
                    self.refs[self.table[r, j]] -= 1
                    self.table[r, j] = -1
                self.lens[r] = keep[r]

    def compact(self):
        live = int((self.refs > 0).sum())
        holes = [p for p in range(live) if self.refs[p] == 0]
        moved = [p for p in range(self.refs.size - 1, live - 1, -1) if self.refs[p] > 0]
        to = np.arange(self.refs.size)
        for s, d in zip(moved, holes):
            self.move(s, d)
            self.refs[d], self.refs[s] = self.refs[s], 0
            to[s] = d
        self.table = np.where(self.table >= 0, to[self.table], self.table).astype(np.int32)
        return live, len(moved)

    def append(self, layer, k, v, start, off):
        rows, page = self.table.shape[0], self.page
        for r in range(rows):
            a, n = int(start[r]), int(off[r + 1] - off[r])
            if a < 0 or n == 0:
                continue
            for b in range(a // 16, -(-(a + n) // 16)):
                lo, hi = max(16 * b, a), min(16 * b + 16, a + n)
                if 16 * b // page >= self.table.shape[1]:
                    continue
                p = self.table[r, 16 * b // page]
                if not 0 <= p < self.refs.size:
                    continue
                at = 16 * b % page
                for x, codes, scales in ((k, self.k, self.ks), (v, self.v, self.vs)):
                    for h in range(codes.shape[2]):
                        new = x[off[r] + lo - a:off[r] + hi - a, h].astype(np.float64)
                        s = scale_for(new)
                        old = codes[layer, p, h, at:at + lo - 16 * b]
                        if lo > 16 * b:
                            had = np.float64(scales[layer, p, h, at // 16])
                            s = max(s, had)
                            old[:] = encode(decode(old) * had / s)
                        codes[layer, p, h, at + lo - 16 * b:at + hi - 16 * b] = encode(new / s)
                        scales[layer, p, h, at // 16] = s


def same(a, b):
    """Codes are equal, NaNs among them by being NaNs."""
    nan = ((a & 0x7F) == 0x7F) & ((b & 0x7F) == 0x7F)
    return bool(((a == b) | nan).all())
