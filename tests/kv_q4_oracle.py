"""The paged 4-bit cache and its attention from their definitions, in numpy and 64 bits."""
from __future__ import annotations

import numpy as np


def as_f64(x: np.ndarray) -> np.ndarray:
    return x.astype(np.float64)


def quantize(x: np.ndarray):
    """[..., D] (any float type, exact in f64) -> codes int [..., D], scales f16 [..., D / 32]."""
    y = as_f64(x).reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    with np.errstate(all="ignore"):
        hi, lo = y.max(-1), y.min(-1)
        m = np.where(hi >= -lo, hi, lo)
        d = np.clip(m / -8.0, -65504.0, 65504.0).astype(np.float32).astype(np.float16)
        finite = np.isfinite(y).all(-1)
        d = np.where(finite, d, np.float16("nan"))
        dd = as_f64(d)[..., None]
        q = np.where((dd == 0) | np.isnan(dd), 0.0, np.round(y / np.where(dd == 0, 1.0, dd)))
        code = np.clip(np.where(np.isnan(q), 0.0, q), -8, 7).astype(np.int64) + 8
    return code.reshape(x.shape), d


def values(code: np.ndarray, d: np.ndarray) -> np.ndarray:
    return ((code.reshape(*d.shape, 32) - 8) * as_f64(d)[..., None]).reshape(code.shape)


class Cache:
    """The bytes of a pool, written and read one value at a time by the layout's definition."""

    def __init__(self, n_pages: int, heads: int, D: int, P: int, fill: int = 0xFF):
        self.n_pages, self.heads, self.D, self.P, self.NB = n_pages, heads, D, P, D // 32
        self.page_bytes = heads * (P // 32) * 36 * D
        self.data = np.full(n_pages * self.page_bytes, fill, np.uint8)

    def cell(self, slot: int, head: int) -> int:
        page, at = divmod(slot, self.P)
        return page * self.page_bytes + (head * (self.P // 32) + at // 32) * 36 * self.D

    def _places(self, value: bool):
        """(byte in the token's cell, shift) of every dim, for token (u, g, i): a function."""
        NB = self.NB

        def of(t):
            u, g, i = t // 16, t % 16 // 4, t % 4
            out = []
            for x in range(self.D):
                b, e = divmod(x, 32)
                if value:
                    word = ((((b // 2) * 16 + e % 16) * 4 + g) * 2 + b % 2) * 2 + u
                    out.append((18 * self.D + 4 * word + i, 4 * (e // 16)))
                else:
                    q, j = divmod(e, 8)
                    nib = j // 2 + 4 * (j % 2)
                    out.append((4 * (((16 * u + 4 * g + i) * 4 + q) * NB + b) + nib // 2, 4 * (nib % 2)))
            base = 34 * self.D if value else 16 * self.D
            scales = [base + 2 * (((4 * u + g) * NB + b) * 4 + i) for b in range(NB)]
            return np.array(out), np.array(scales)
        return [of(t) for t in range(32)]

    def tables(self):
        if not hasattr(self, "_tab"):
            self._tab = (self._places(False), self._places(True))
        return self._tab

    def store(self, k, v, slots):
        for x, tab in zip((k, v), self.tables()):
            code, d = quantize(x)
            for r, s in enumerate(slots):
                if s < 0:
                    continue
                place, scales = tab[s % self.P % 32]
                for h in range(self.heads):
                    c = self.cell(int(s), h)
                    at, sh = c + place[:, 0], place[:, 1]
                    for half in (0, 4):
                        m = sh == half
                        self.data[at[m]] = (self.data[at[m]] & (0xF0 if half == 0 else 0x0F)) | (code[r, h][m] << half).astype(np.uint8)
                    for b in range(self.NB):
                        self.data[c + scales[b]:c + scales[b] + 2] = np.frombuffer(d[r, h, b].tobytes(), np.uint8)

    def load(self, slots):
        """f64 (k, v) [rows, heads, D]."""
        out = []
        for tab in self.tables():
            o = np.zeros((len(slots), self.heads, self.D))
            for r, s in enumerate(slots):
                place, scales = tab[int(s) % self.P % 32]
                for h in range(self.heads):
                    c = self.cell(int(s), h)
                    code = (self.data[c + place[:, 0]].astype(np.int64) >> place[:, 1]) & 15
                    d = np.array([np.frombuffer(self.data[c + a:c + a + 2].tobytes(), np.float16)[0] for a in scales])
                    o[r, h] = values(code, d)
            out.append(o)
        return tuple(out)


def attention(q, k, v, n: int, scale: float):
    """q [n, Hq, D], k, v [len, Hk, D] in f64 -> (out, sum of p |v|, largest sum of |q k| scale, p's largest share)."""
    Hq, Hk, D = q.shape[1], k.shape[1], q.shape[2]
    out, mag, big = np.zeros((n, Hq, D)), np.zeros((n, Hq, D)), np.zeros((n, Hq, 1))
    length = k.shape[0]
    for t in range(n):
        seen = length - n + t + 1
        if seen <= 0:
            continue
        for h in range(Hq):
            g = h // (Hq // Hk)
            with np.errstate(invalid="ignore", over="ignore"):
                s = k[:seen, g] @ q[t, h] * scale
                p = np.exp(s - s.max())
                p = p / p.sum()
                out[t, h] = p @ v[:seen, g]
                mag[t, h] = p @ np.abs(v[:seen, g])
                big[t, h] = (np.abs(k[:seen, g]) @ np.abs(q[t, h]) * scale).max()
    return out, mag, big


def plan(held, past, new, P, table, ring, counters, T):
    """The bookkeeping, request by request; table and ring are changed.  Returns (counters, start, lens, slot, pos, status)."""
    S, W = table.shape
    N = len(ring)
    head, tail = int(counters[0]), int(counters[1])
    avail = max(0, min(tail - head, N))
    start, lens, slot, pos, status = [0], [], [-1] * T, [-1] * T, 0
    wanted = taken = given = 0
    for i in range(S):
        h, p, n = int(held[i]), int(past[i]), int(new[i])
        at, end = start[-1], start[-1] + max(n, 0)
        have, need = -(-h // P), -(-(p + max(n, 0)) // P)
        ok = h >= 0 and 0 <= p <= h and n >= 0 and have <= W and need <= W and end <= T
        start.append(end)
        if not ok:
            status |= 32
            lens.append(0)
            continue
        wanted += max(0, need - have)
        if need > have and wanted > avail:
            status |= 16
            lens.append(0)
            continue
        for c in range(have, need):
            table[i, c] = ring[(head + taken) % N]
            taken += 1
        for c in range(need, have):
            ring[(tail + given) % N] = table[i, c]
            given += 1
        for r in range(n):
            x = p + r
            page = int(table[i, x // P])
            if 0 <= page < N:
                slot[at + r] = page * P + x % P
            else:
                status |= 4
            pos[at + r] = x
        lens.append(p + n)
    return (np.array([head + taken, tail + given]), np.minimum(start, T), np.array(lens), np.array(slot), np.array(pos), status)
