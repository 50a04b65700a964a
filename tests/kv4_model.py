"""The 4-bit KV format and its attention in 64 bits (numpy), written from the
definitions in include/axkv.h, and the page table as plain Python lists."""
from __future__ import annotations

import numpy as np

LIMIT = 32768.0


def steps() -> np.ndarray:
    """Every fp16 number with the low 4 mantissa bits clear, ascending from 0."""
    return (np.arange(0x7C0, dtype=np.uint16) << 4).view(np.float16).astype(np.float64)


def quantize(x: np.ndarray):
    """x [..., 32 m] fp32 -> q [..., 32 m], code and z [..., m]."""
    b = np.nan_to_num(x.astype(np.float64), nan=0.0, posinf=LIMIT, neginf=-LIMIT)
    b = np.clip(b, -LIMIT, LIMIT).reshape(*x.shape[:-1], -1, 32)
    lo, hi = np.minimum(b.min(-1), 0), np.maximum(b.max(-1), 0)
    R = (hi.astype(np.float32) - lo.astype(np.float32)).astype(np.float64)
    code = np.searchsorted(15 * steps(), R)
    d = np.where(code == 0, 1.0, steps()[code])[..., None]
    z = -np.floor(lo[..., None] / d + 0.5)
    q = np.minimum(np.floor(b / d + 0.5) + z, 15)
    assert q.min() >= 0 and z.min() >= 0 and z.max() <= 15
    return q.astype(np.int64).reshape(x.shape), code, z[..., 0].astype(np.int64)


def values(x: np.ndarray) -> np.ndarray:
    """What the cache holds for x, in 64 bits."""
    q, code, z = quantize(x)
    b = q.reshape(*code.shape, 32) - z[..., None]
    return (steps()[code][..., None] * b).reshape(x.shape)


def write_token(page: np.ndarray, slot: int, k: np.ndarray, v: np.ndarray) -> None:
    """One token's K and V (k, v [hd]) into the bytes of a (page, head): the layout, byte by byte."""
    hd = k.shape[0]
    nb, tpg = hd // 32, min(4, hd // 16)
    for part, x in ((0, k), (1, v)):
        q, code, z = quantize(x)
        for b in range(nb):
            w = int(code[b]) << 4 | int(z[b])
            at = (16 + part) * hd + (slot * nb + b) * 2
            page[at], page[at + 1] = w & 255, w >> 8
        for dim in range(hd):
            if part == 0:
                b, t, e = dim // 32, dim % 32 // 8, dim % 8
                at, high = slot * (hd // 2) + t * (hd // 8) + 4 * b + e // 2, e % 2
            else:
                tile, g, high = dim // 16, dim % 8, dim % 16 // 8
                u, t, w = slot % 2, slot % 8 // 2, slot // 8
                at = 8 * hd + tile // tpg * 128 * tpg + ((g * 4 + t) * tpg + tile % tpg) * 4 + 2 * u + w
            page[at] = (int(page[at]) & (15 if high else 240)) | int(q[dim]) << (4 if high else 0)


def attention(q: np.ndarray, k: np.ndarray, v: np.ndarray, scale: float) -> np.ndarray:
    """q [hd], k, v [n, hd] in 64 bits; no token: zeros."""
    if len(k) == 0:
        return np.zeros(v.shape[-1])
    s = (k @ q) * scale
    p = np.exp(s - s.max())
    return p @ v / p.sum()


def tolerance(q: np.ndarray, k: np.ndarray, v: np.ndarray, scale: float) -> float:
    """How far an fp32 result may be: scores carry at most (hd + 8) rounding steps of
    2^-24 of sum |q k| (the fp16 pairs of q add 2^-22 of it, within the 8), weights
    twice that and their own roundings, and sums of n terms n steps each, numerator and
    denominator; all relative to the largest value."""
    if len(k) == 0:
        return 0.0
    ds = scale * (q.shape[-1] + 8) * 2.0 ** -24 * (np.abs(k) @ np.abs(q)).max()
    return float((2 * ds + (2 * len(k) + 32) * 2.0 ** -24) * np.abs(v).max())


class Table:
    """Block table and counts; each call as the header defines it, or None where it is refused."""

    def __init__(self, n_seqs: int, max_blocks: int, n_pages: int):
        self.rows = [[] for _ in range(n_seqs)]
        self.max_blocks, self.n_pages = max_blocks, n_pages

    def counts(self) -> np.ndarray:
        c = np.zeros(self.n_pages, np.int32)
        for r in self.rows:
            for p in r:
                c[p] += 1
        return c

    def array(self) -> np.ndarray:
        t = np.full((len(self.rows), self.max_blocks), -1, np.int32)
        for i, r in enumerate(self.rows):
            t[i, :len(r)] = r
        return t

    def _free(self) -> list[int]:
        return [int(i) for i in np.nonzero(self.counts() == 0)[0]]

    def reserve(self, seqs, tokens):
        if len(set(seqs)) < len(seqs) or any(not 0 <= s < len(self.rows) for s in seqs) \
                or any(not 0 <= t <= 16 * self.max_blocks for t in tokens):
            return None
        need = [max(0, -(-t // 16) - len(self.rows[s])) for s, t in zip(seqs, tokens)]
        free = self._free()
        if sum(need) > len(free):
            return None
        for s, n in zip(seqs, need):
            self.rows[s] += free[:n]
            free = free[n:]
        return True

    def fork(self, parents, children, tokens):
        n = len(self.rows)
        if len(set(children)) < len(children) or set(parents) & set(children) \
                or any(not 0 <= s < n for s in list(parents) + list(children)) \
                or any(self.rows[c] for c in children) \
                or any(not 0 <= t <= 16 * len(self.rows[p]) for p, t in zip(parents, tokens)):
            return None
        free = self._free()
        copies = []
        if sum(t % 16 > 0 for t in tokens) > len(free):
            return None
        for p, c, t in zip(parents, children, tokens):
            self.rows[c] = self.rows[p][:t // 16]
            if t % 16:
                copies.append((self.rows[p][t // 16], free[0]))
                self.rows[c] = self.rows[c] + [free.pop(0)]
        return copies

    def free(self, seqs):
        for s in seqs:
            if 0 <= s < len(self.rows):
                self.rows[s] = []

    def compact(self):
        c = self.counts()
        live = int((c > 0).sum())
        src = [i for i in range(live, self.n_pages) if c[i]]
        dst = [i for i in range(live) if not c[i]]
        to = dict(zip(src, dst))
        self.rows = [[to.get(p, p) for p in r] for r in self.rows]
        return live, list(zip(src, dst))
