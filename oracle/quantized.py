"""CPU oracle of the 8-bit KV cache (test infrastructure only): the append's
scale rule code by code, attention in 64 bits from its definition, and the
eviction row by row."""

from __future__ import annotations

import math
from dataclasses import dataclass

import numpy as np

from oracle import numerics as nm

D = 128
U = 2.0 ** -24  # half a step of a float32 at 1


def block_scale(amax: float) -> float:
    """The smallest power of two s >= 2^-64 with amax <= 448 s."""
    s = 2.0 ** -64
    while amax > 448.0 * s:
        s *= 2.0
    return s


def encode(x: np.ndarray) -> np.ndarray:
    """E4M3 codes, nearest even; what is not finite becomes NaN (0x7f)."""
    return np.where(np.isfinite(x), nm.f32_to_e4m3(np.where(np.isfinite(x), x, 0)), np.uint8(0x7F)).astype(np.uint8)


def decode(codes: np.ndarray) -> np.ndarray:
    return nm.e4m3_to_f32(codes).astype(np.float64)


@dataclass
class Cache:
    codes: list          # keys, values: uint8 [B, H, C, 128]
    scales: list         # float32 [B, H, C / block]
    positions: np.ndarray
    weights: np.ndarray  # float32 [B, H, C]
    cursors: np.ndarray  # int32 [3, B]
    block: int

    @classmethod
    def of(cls, cache) -> "Cache":
        """A copy of a device cache."""
        import torch

        def host(t):
            return t.cpu().numpy().copy()

        weights = torch.zeros_like(cache.positions, dtype=torch.float32) if cache.weights is None else cache.weights
        return cls([host(cache.key_codes.view(torch.uint8)), host(cache.value_codes.view(torch.uint8))],
                   [host(cache.key_scales), host(cache.value_scales)], host(cache.positions), host(weights),
                   host(cache.cursors), cache.block)

    @property
    def capacity(self) -> int:
        return self.positions.shape[2]

    def value(self, tensor: int, b: int, h: int, rows) -> np.ndarray:
        rows = np.asarray(rows, dtype=np.int64)
        scale = self.scales[tensor][b, h, rows // self.block].astype(np.float64)
        return decode(self.codes[tensor][b, h, rows]) * scale[:, None]

    def put(self, tensor: int, b: int, h: int, blk: int, rows, values: np.ndarray, before) -> None:
        """Writes `values` (exact, 64 bits) into rows of block `blk`; `before`
        are the block's rows that were there and stay."""
        finite = np.abs(values[np.isfinite(values)])
        need = block_scale(float(finite.max()) if finite.size else 0.0)
        old = float(self.scales[tensor][b, h, blk]) if before is not None else 0.0
        scale = max(old, need)
        if before is not None and scale != old and len(before):
            stay = self.codes[tensor][b, h, before]
            self.codes[tensor][b, h, before] = encode(decode(stay) * (old / scale))
        self.scales[tensor][b, h, blk] = scale
        self.codes[tensor][b, h, rows] = encode(values / scale)

    def append(self, key: np.ndarray, value: np.ndarray, counts=None) -> None:
        """key, value: float64 [B, H, T, 128]."""
        batch, heads, tokens, _ = key.shape
        for b in range(batch):
            count = tokens if counts is None else min(max(int(counts[b]), 0), tokens)
            start, seen = int(self.cursors[0, b]), int(self.cursors[1, b])
            end = min(start + count, self.capacity)
            for h in range(heads):
                for tensor, x in ((0, key), (1, value)):
                    row = start
                    while row < end:
                        blk = row // self.block
                        stop = min(end, (blk + 1) * self.block)
                        before = np.arange(blk * self.block, start) if blk * self.block < start else None
                        self.put(tensor, b, h, blk, np.arange(row, stop), x[b, h, row - start:stop - start], before)
                        row = stop
                self.positions[b, h, start:end] = seen + np.arange(end - start)
                self.weights[b, h, start:end] = 0
            if start + count > self.capacity:
                self.cursors[2, b] = 1
            self.cursors[0, b], self.cursors[1, b] = end, seen + end - start

    def attend(self, query: np.ndarray, *, scale: float, counts=None, window: int = 0, pieces: int = 1, half_step=2.0 ** -8):
        """query float64 [B, Hq, T, 128].  Returns out [B, T, Hq, D], lse
        [B, Hq, T], received [B, H, C], and how far a kernel may be from each:

        a score is a sum of 128 products of exact factors for each of the
        `pieces` bf16 pieces of the query, added in 32 bits (the matrix core may
        round a sum either way, by a whole step 2 u, u = 2^-24) and multiplied
        by rounded factors, so it is off by at most
        d = (256 pieces + 4) u scale sum|q k|; a probability is then off by the
        factor e^(2 d) (its own score and the sum's), four roundings of the
        exponential and the division, and the n additions of the sum; the value
        product takes it rounded to `pieces` bf16 pieces (2^-8 each) and adds
        n `pieces` terms; the result is rounded to its type (half a step).
        Underflow to zero loses less than 2^-126 of a row's weight."""
        batch, hq, tokens, _ = query.shape
        heads = self.positions.shape[1]
        group = hq // heads
        out = np.zeros((batch, tokens, hq, D))
        out_tol = np.zeros_like(out)
        lse = np.full((batch, hq, tokens), -np.inf)
        lse_tol = np.zeros_like(lse)
        got = np.zeros(self.positions.shape)
        got_tol = np.zeros_like(got)
        for b in range(batch):
            n, seen = int(self.cursors[0, b]), int(self.cursors[1, b])
            count = tokens if counts is None else min(max(int(counts[b]), 0), tokens)
            for h in range(heads):
                k, v = self.value(0, b, h, np.arange(n)), self.value(1, b, h, np.arange(n))
                pos = self.positions[b, h, :n].astype(np.int64)
                for t in range(count):
                    at = seen - count + t
                    rows = np.flatnonzero((pos <= at) & ((pos > at - window) if window else True))
                    if not rows.size:
                        continue
                    for g in range(h * group, (h + 1) * group):
                        q = query[b, g, t]
                        s = (k[rows] @ q) * scale
                        d = (256 * pieces + 4) * U * scale * float((np.abs(k[rows]) @ np.abs(q)).max())
                        top = s.max()
                        p = np.exp(s - top)
                        z = p.sum()
                        share = p / z
                        out[b, t, g] = share @ v[rows]
                        size = share @ np.abs(v[rows])
                        loose = math.expm1(2 * d) + (rows.size + 8) * U
                        out_tol[b, t, g] = (half_step * np.abs(out[b, t, g]) +
                                            (1 + half_step) * size * (loose + (2.0 ** -8) ** pieces + 2 * rows.size * pieces * U))
                        lse[b, g, t] = top + math.log(z)
                        lse_tol[b, g, t] = d + (rows.size + 8) * U + 4 * U * (abs(lse[b, g, t]) + abs(top))
                        got[b, h, rows] += share
                        got_tol[b, h, rows] += share * (loose + (group * count + 4) * U) + 1e-37
        return (out, lse, got), (out_tol, lse_tol, got_tol)

    def evict(self, *, keep: int, num_sink: int = 0, recent: int = 0, into: "Cache | None" = None) -> None:
        source = Cache([c.copy() for c in self.codes], [s.copy() for s in self.scales], self.positions.copy(),
                       self.weights.copy(), self.cursors.copy(), self.block)
        to = self if into is None else into
        batch, heads, _ = self.positions.shape
        for b in range(batch):
            n, seen = int(source.cursors[0, b]), int(source.cursors[1, b])
            left = min(n, keep)
            for h in range(heads):
                def order(r):
                    p, w = int(source.positions[b, h, r]), float(source.weights[b, h, r])
                    if p < num_sink or p >= seen - recent:
                        return (0, 0.0, r)
                    return (1, 0.0, r) if math.isnan(w) else (2, -w, r)

                kept = set(sorted(range(n), key=order)[:keep]) if n > keep else set(range(n))
                holes = [r for r in range(left) if r not in kept]
                movers = sorted(r for r in kept if r >= left)
                assert len(holes) == len(movers)
                comes = dict(zip(holes, movers))
                for blk in range(-(-left // self.block)):
                    rows = range(blk * self.block, min((blk + 1) * self.block, left))
                    stay = np.array([r for r in rows if r not in comes], dtype=np.int64)
                    moved = np.array([r for r in rows if r in comes], dtype=np.int64)
                    for tensor in (0, 1):
                        if into is not None:
                            to.codes[tensor][b, h, stay] = source.codes[tensor][b, h, stay]
                            to.scales[tensor][b, h, blk] = source.scales[tensor][b, h, blk]
                        if moved.size:
                            values = source.value(tensor, b, h, [comes[r] for r in moved])
                            to.put(tensor, b, h, blk, moved, values, stay)
                for r in range(left):
                    m = comes.get(r, r)
                    to.positions[b, h, r] = source.positions[b, h, m]
                    to.weights[b, h, r] = source.weights[b, h, m]
            to.cursors[0, b] = left
            to.cursors[1:, b] = source.cursors[1:, b]
