"""The 4-bit token cache in plain numpy, 64 bits: format, pages, attention.

Test infrastructure only, written from the format's definition: a code is a sign
bit, two exponent bits E and a mantissa bit M, of magnitude M / 2 where E = 0 and
2^(E - 1) * (1 + M / 2) otherwise; 32 dims share a scale byte s = 2^(s - 127), the
smallest power of two under which none of them passes 6; a value takes the nearest
code, between two the one with M = 0; a block with a NaN or an infinity has scale
byte 255 and reads as NaN.  Pinned by hand-worked codes and by the nearest of all
sixteen values (tests/test_oracle_fp4.py).
"""

from __future__ import annotations

import numpy as np

BLOCK = 32
LEVELS = np.array([0.5 * (c & 1) if c < 2 else 2.0 ** ((c >> 1) - 1) * (1 + 0.5 * (c & 1)) for c in range(8)])


def quantize(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """Codes (uint8 0..15) of x [..., D] and scale bytes [..., D / 32]."""
    b = np.asarray(x, dtype=np.float64).reshape(*x.shape[:-1], -1, BLOCK)
    bad = ~np.isfinite(b).all(-1)
    big = np.where(bad, 0.0, np.abs(np.where(np.isfinite(b), b, 0.0)).max(-1))
    e = np.full(big.shape, -120, dtype=np.int64)
    for k in range(-120, 125):  # the smallest exponent that is large enough
        e = np.where(6.0 * 2.0 ** k < big, k + 1, e)
    a = np.where(bad[..., None], 0.0, b) / 2.0 ** e[..., None]
    mag = np.minimum(np.abs(a), 6.0)
    code = np.zeros(a.shape, dtype=np.int64)
    for c in range(1, 8):
        mid = (LEVELS[c] + LEVELS[c - 1]) / 2
        code = np.where((mag > mid) | ((mag == mid) & (c % 2 == 0)), c, code)
    code = np.where(bad[..., None], 0, code + 8 * np.signbit(a))
    byte = np.where(bad, 255, e + 127)
    return code.reshape(x.shape).astype(np.uint8), byte.astype(np.uint8)


def dequantize(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """Values of codes [..., D] under scale bytes [..., D / 32]."""
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    v = np.where(codes >= 8, -1.0, 1.0) * LEVELS[codes & 7]
    return v * np.repeat(s, BLOCK, axis=-1)


class Pages:
    """A pool of pages as bytes [n_pages, block, heads, 17 * dim / 16], and access
    to a token's codes and scale bytes in it."""

    def __init__(self, pool: np.ndarray) -> None:
        self.pool = pool
        self.n_pages, self.block, self.heads, row = pool.shape
        self.dim = row * 16 // 17
        self.flat = pool.reshape(self.n_pages, self.heads, -1)

    def _at(self, slot: int, kv: int) -> tuple[slice, slice]:
        half, row, nb = self.block * self.dim // 2, self.dim // 2, self.dim // BLOCK
        c = kv * half + slot * row
        s = 2 * half + (2 * slot + kv) * nb
        return slice(c, c + row), slice(s, s + nb)

    def write(self, page: int, slot: int, kv: int, x: np.ndarray) -> None:
        """x [heads, dim] becomes token `slot` of the page."""
        codes, scales = quantize(x)
        c, s = self._at(slot, kv)
        self.flat[page, :, c] = codes[:, 0::2] + 16 * codes[:, 1::2]
        self.flat[page, :, s] = scales

    def read(self, page: int, slot: int, kv: int) -> np.ndarray:
        c, s = self._at(slot, kv)
        b = self.flat[page, :, c]
        codes = np.stack([b & 15, b >> 4], axis=-1).reshape(self.heads, self.dim)
        return dequantize(codes, self.flat[page, :, s])


def append(pool: np.ndarray, block_table: np.ndarray, seq_lens: np.ndarray, k: np.ndarray, v: np.ndarray,
           n_new: np.ndarray) -> None:
    """The n_new[b] newest tokens of each sequence (seq_lens counts them) from k, v [B, T, heads, dim]."""
    p = Pages(pool)
    for b in range(block_table.shape[0]):
        for i in range(int(n_new[b])):
            pos = int(seq_lens[b]) - int(n_new[b]) + i
            for kv, x in enumerate((k, v)):
                p.write(int(block_table[b, pos // p.block]), pos % p.block, kv, x[b, i])


def rows(pool: np.ndarray, block_table: np.ndarray, b: int, positions: range) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
    """Keys and values [n, heads, dim] of a sequence's positions, and which pages are mapped."""
    p = Pages(pool)
    k = np.zeros((len(positions), p.heads, p.dim))
    v, mapped = np.zeros_like(k), np.zeros(len(positions), dtype=bool)
    for i, pos in enumerate(positions):
        page = int(block_table[b, pos // p.block])
        if 0 <= page < p.n_pages:
            k[i], v[i], mapped[i] = p.read(page, pos % p.block, 0), p.read(page, pos % p.block, 1), True
    return k, v, mapped


def attention(q: np.ndarray, pool: np.ndarray, block_table: np.ndarray, seq_lens: np.ndarray, window: int | None = None,
              sink: np.ndarray | None = None, softcap: float | None = None, scale: float | None = None,
              n_new: np.ndarray | None = None) -> np.ndarray:
    """q [B, T, H, D] over the pages, one (token, head) at a time; of sequence b the first n_new[b] tokens."""
    batch, t_new, heads, dim = q.shape
    out = np.zeros(q.shape)
    for b in range(batch):
        length = int(seq_lens[b])
        k, v, mapped = rows(pool, block_table, b, range(length))
        own = t_new if n_new is None else min(int(n_new[b]), t_new)
        for t in range(own):
            end = length - own + t + 1
            begin = max(0, end - window) if window else 0
            live = np.flatnonzero(mapped[begin:max(end, 0)]) + begin if end > 0 else np.zeros(0, dtype=np.int64)
            if live.size == 0:
                continue
            for h in range(heads):
                hk = h // (heads // k.shape[1])
                kk, vv = k[live, hk], v[live, hk]
                if np.isnan(vv).any():  # a NaN among the values is seen whole
                    out[b, t, h] = np.nan
                    continue
                s = kk @ q[b, t, h].astype(np.float64) * (dim ** -0.5 if scale is None else scale)
                if softcap:
                    s = softcap * np.tanh(s / softcap)
                top = s.max() if sink is None else max(s.max(), float(sink[h]))
                w = np.exp(s - top)
                out[b, t, h] = w @ vv / (w.sum() + (0.0 if sink is None else np.exp(float(sink[h]) - top)))
    return out


def ancestors(parents: list[int], t: int) -> list[int] | None:
    """Node t's ancestors and itself, ascending, or None where a parent on the way up is not an earlier node (-1: none)."""
    got = []
    while t != -1:
        got.append(t)
        if not -1 <= parents[t] < t:
            return None
        t = parents[t]
    return got[::-1]


def tree_masks(parents: np.ndarray, n_new: np.ndarray) -> np.ndarray:
    """bool [B, T, T]: node t sees node j (itself, its ancestors); none of a node past n_new[b] or with a bad parent."""
    batch, t_max = parents.shape
    seen = np.zeros((batch, t_max, t_max), dtype=bool)
    for b in range(batch):
        for t in range(min(int(n_new[b]), t_max)):
            up = ancestors([int(p) for p in parents[b]], t)
            if up is not None:
                seen[b, t, up] = True
    return seen


def pack_masks(seen: np.ndarray) -> np.ndarray:
    """bool [B, T, T] to int64 [B, T, ceil(T / 64)], bit j % 64 of word j / 64."""
    t = seen.shape[2]
    wide = np.zeros((*seen.shape[:2], -(-t // 64) * 64), dtype=np.uint64)
    wide[..., :t] = seen
    words = wide.reshape(*seen.shape[:2], -1, 64) << np.arange(64, dtype=np.uint64)
    return np.bitwise_or.reduce(words, axis=-1).view(np.int64)


def history(length: int, own: int, t: int, seen: np.ndarray | None) -> list[int]:
    """The positions of token t's history: those before the `own` new tokens, then the new ones that it sees (`seen`, a
    row of masks; None: those up to itself)."""
    base = length - own
    if seen is None:
        return list(range(max(base + t + 1, 0)))
    new = [j for j in range(t + 1) if seen[j]]
    return list(range(base)) + [base + j for j in new] if new and base >= 0 else []


def view_attention(q: np.ndarray, pool: np.ndarray, block_table: np.ndarray, seq_lens: np.ndarray, *, window: int | None = None,
                   first: int = 0, seen: np.ndarray | None = None, sink: np.ndarray | None = None,
                   softcap: float | None = None, scale: float | None = None, n_new: np.ndarray | None = None) -> np.ndarray:
    """As ``attention`` where a token sees the last `window` and the first `first` positions of its history."""
    batch, t_new, heads, dim = q.shape
    out = np.zeros(q.shape)
    for b in range(batch):
        length = int(seq_lens[b])
        k, v, mapped = rows(pool, block_table, b, range(length))
        own = t_new if n_new is None else min(int(n_new[b]), t_new)
        for t in range(own):
            hist = history(length, own, t, None if seen is None else seen[b, t])
            if window:
                hist = [p for i, p in enumerate(hist) if i < first or i >= len(hist) - window]
            live = np.array([p for p in hist if mapped[p]], dtype=np.int64)
            if live.size == 0:
                continue
            for h in range(heads):
                hk = h // (heads // k.shape[1])
                kk, vv = k[live, hk], v[live, hk]
                if np.isnan(vv).any():
                    out[b, t, h] = np.nan
                    continue
                s = kk @ q[b, t, h].astype(np.float64) * (dim ** -0.5 if scale is None else scale)
                if softcap:
                    s = softcap * np.tanh(s / softcap)
                top = s.max() if sink is None else max(s.max(), float(sink[h]))
                w = np.exp(s - top)
                out[b, t, h] = w @ vv / (w.sum() + (0.0 if sink is None else np.exp(float(sink[h]) - top)))
    return out
