"""Paged KV cache and drafted trees in 64 bits, row by row (test infrastructure only).

State is plain numpy: pages [layers, pages, heads, page, 128] float64, a page
table and lengths.  Written from the definitions, with no code of the package.
"""

from __future__ import annotations

import math

import numpy as np

D = 128
U = 2.0 ** -24


def tree_of(parents, count):
    """Depths and ancestor sets (lists of lists) of one sequence's first `count` tokens."""
    kin = []
    for t in range(count):
        p = int(parents[t])
        kin.append((kin[p] if 0 <= p < t else []) + [t])
    return [len(k) - 1 for k in kin], kin


def plan(parents, counts=None):
    """Depths [B, T] int32 and masks [B, T, words] int64."""
    batch, tokens = parents.shape
    depths = np.zeros((batch, tokens), np.int32)
    masks = np.zeros((batch, tokens, -(-tokens // 64)), np.uint64)
    for b in range(batch):
        count = tokens if counts is None else min(max(int(counts[b]), 0), tokens)
        d, kin = tree_of(parents[b], count)
        depths[b, :count] = d
        for t, ancestors in enumerate(kin):
            for j in ancestors:
                masks[b, t, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return depths, masks.view(np.int64)


class Paged:
    def __init__(self, keys, values, table, lengths):
        self.keys, self.values = keys.copy(), values.copy()
        self.table, self.lengths = table.copy(), lengths.copy()
        self.page = keys.shape[3]
        self.overflow = np.zeros(len(lengths), np.int32)

    @property
    def capacity(self):
        return self.table.shape[1] * self.page

    @classmethod
    def of(cls, cache):
        keys, values = (t.cpu().double().numpy() for t in (cache.key_pages, cache.value_pages))
        state = cls(keys, values, cache.page_table.cpu().numpy(), cache.lengths.cpu().numpy())
        state.overflow = cache.overflow.cpu().numpy().copy()  # a flag stays until its owner clears it
        return state

    def place(self, b, row):
        """Page and offset of a row, or None."""
        if row >= self.capacity:
            return None
        page = int(self.table[b, row // self.page])
        return (page, row % self.page) if 0 <= page < self.keys.shape[1] else None

    def _start(self, b):
        return min(max(int(self.lengths[b]), 0), self.capacity)

    @staticmethod
    def _steps(tokens, parents, counts, b):
        count = tokens if counts is None else min(max(int(counts[b]), 0), tokens)
        return tree_of(range(-1, count - 1) if parents is None else parents[b], count)

    @staticmethod
    def turn(x, cosines, sines, interleaved):
        """x [..., 128] turned by one position's angles."""
        half = len(cosines)
        out = x.copy()
        for i in range(half):
            p, q = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
            out[..., p] = x[..., p] * cosines[i] - x[..., q] * sines[i]
            out[..., q] = x[..., q] * cosines[i] + x[..., p] * sines[i]
        return out

    def append(self, layer, key, value, query=None, table=None, interleaved=False, parents=None, counts=None):
        """key/value/query float64 [B, H, T, 128]; table (cosines, sines) float64.  Writes unrounded values; returns the
        turned queries, zeros past the counts, and which pages' rows were written."""
        batch, _, tokens, _ = key.shape
        written = np.zeros(self.keys.shape[1:4], bool)
        turned = None if query is None else np.zeros_like(query)
        for b in range(batch):
            depths, _ = self._steps(tokens, parents, counts, b)
            for t, depth in enumerate(depths):
                at = min(self._start(b) + depth, 1 << 30)
                k = key[b, :, t]
                if table is not None:
                    angles = (table[0][min(at, len(table[0]) - 1)], table[1][min(at, len(table[1]) - 1)])
                    k = self.turn(k, *angles, interleaved)
                    if query is not None:
                        turned[b, :, t] = self.turn(query[b, :, t], *angles, interleaved)
                place = self.place(b, self._start(b) + t)
                if place is None:
                    self.overflow[b] = 1
                    continue
                self.keys[layer, place[0], :, place[1]] = k
                self.values[layer, place[0], :, place[1]] = value[b, :, t]
                written[place[0], :, place[1]] = True
        return turned, written

    def sees(self, b, t, depths, kin, window):
        """Rows that token t sees, in order."""
        start = self._start(b)
        low = start + depths[t] - window + 1 if window else 0
        rows = [r for r in range(max(low, 0), start)]
        rows += [start + j for j in kin[t] if start + depths[j] >= low]
        return [r for r in rows if self.place(b, r) is not None]

    def attend(self, layer, query, *, scale, parents=None, counts=None, window=0, half_step=2.0 ** -8):
        """query float64 [B, Hq, T, 128].  Returns out [B, T, Hq, 128], lse [B, Hq, T] and how far a kernel may be from each.

        A score is a sum of 128 products of exact factors added in 32 bits (the matrix core may round a sum either way, by a
        whole step 2 u, u = 2^-24) and multiplied by rounded factors: off by at most d = (256 + 4) u scale sum|q k|.  A
        probability is off by the factor e^(2 d) (its own score and the sum's), four roundings of the exponential and the
        division, the argument of the exponential (off by 2 u of a few hundreds, in log2 units: |s| log2(e) 2 u more), and the n
        additions of the sum; the value product takes it rounded to the type (half_step of it; fp16 ones are kept 2^7 as large,
        so what lies below their normal range is off by at most 2^-25 of 2^7, that is 2^-32 of the sum at most per row) and adds n
        terms; parts are joined with two roundings more each; the result is rounded to the type.  Underflow to zero loses less
        than 2^-126 of a row's weight."""
        batch, hq, tokens, _ = query.shape
        heads = self.keys.shape[2]
        group = hq // heads
        out = np.zeros((batch, tokens, hq, D))
        lse = np.full((batch, hq, tokens), -np.inf)
        out_tol, lse_tol = np.zeros_like(out), np.zeros_like(lse)
        for b in range(batch):
            depths, kin = self._steps(tokens, parents, counts, b)
            for t in range(len(depths)):
                rows = self.sees(b, t, depths, kin, window)
                if not rows:
                    continue
                places = [self.place(b, r) for r in rows]
                pages, offsets = np.array([p for p, _ in places]), np.array([o for _, o in places])
                for h in range(heads):
                    k, v = self.keys[layer, pages, h, offsets], self.values[layer, pages, h, offsets]
                    q = query[b, h * group:(h + 1) * group, t]
                    s = (q @ k.T) * scale
                    d = 260 * U * scale * (np.abs(q) @ np.abs(k).T).max(1)
                    top = s.max(1)
                    p = np.exp(s - top[:, None])
                    z = p.sum(1)
                    share = p / z[:, None]
                    o, size = share @ v, share @ np.abs(v)
                    loose = np.expm1(2 * d) + (len(rows) + 16) * U + 6 * U * np.abs(s).max(1)
                    most = np.abs(v).max() if half_step < 2.0 ** -8 else 0.0
                    at = slice(h * group, (h + 1) * group)
                    out[b, t, at] = o
                    out_tol[b, t, at] = (half_step * np.abs(o) + 2.0 ** -25 +
                                         (1 + half_step) * size * (loose + half_step + 2 * len(rows) * U)[:, None] +
                                         len(rows) * 2.0 ** -32 * most)
                    lse[b, at, t] = top + np.log(z)
                    lse_tol[b, at, t] = d + (len(rows) + 16) * U + 6 * U * (np.abs(lse[b, at, t]) + np.abs(s).max(1))
        return (out, lse), (out_tol, lse_tol)

    def commit(self, counts, path=None):
        for b in range(len(self.lengths)):
            start = self._start(b)
            room = self.capacity - start
            count = max(int(counts if np.isscalar(counts) else counts[b]), 0)
            if path is None:
                self.lengths[b] = start + min(count, room)
                continue
            kept = []
            for p in path[b][:count]:
                if p >= room or p <= (kept[-1] if kept else -1):
                    break
                kept.append(int(p))
            for j, p in enumerate(kept):
                to, source = self.place(b, start + j), self.place(b, start + p)
                if to is None or source is None:
                    continue
                for pages in (self.keys, self.values):
                    pages[:, to[0], :, to[1]] = pages[:, source[0], :, source[1]]
            self.lengths[b] = start + len(kept)
