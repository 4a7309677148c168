"""Oracle of the paged KV cache in 64 bits: rotation, what each cache type holds of a row, pages, and attention with a window and first tokens.
Shares no code with the product."""
from __future__ import annotations

import numpy as np


def quantize_q4_0(x):
    """Q4_0 of fp32 values in blocks of 32 along the last axis (gguf-py 0.19.0, Q4_0.quantize_blocks): (q uint8 [..., n], d float16 [..., n / 32])"""
    x = np.ascontiguousarray(x, dtype=np.float32)
    b = x.reshape(-1, 32)
    m = np.take_along_axis(b, np.abs(b).argmax(axis=1)[:, None], axis=1)
    d = (m / np.float32(-8)).astype(np.float32)
    with np.errstate(all="ignore"):
        inv = np.where(d == 0, np.float32(0), np.float32(1) / d).astype(np.float32)
        q = np.trunc(b.astype(np.float64) * inv.astype(np.float64) + 8.5)
        dh = d.astype(np.float16)
    return np.clip(q, 0, 15).astype(np.uint8).reshape(x.shape), dh.reshape(x.shape[:-1] + (x.shape[-1] // 32,))


def held(x, dtype):
    """what a cache of this type hands back for fp32 rows, as fp64"""
    x = np.asarray(x, dtype=np.float32)
    if dtype == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16).astype(np.float64)
    if dtype == "bf16":
        u = np.ascontiguousarray(x).view(np.uint32)
        r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16 << 16).view(np.float32)
        return np.where(np.isfinite(x), r, x).astype(np.float64)
    q, d = quantize_q4_0(x)
    return (q.astype(np.float64).reshape(-1, 32) - 8).reshape(x.shape) * np.repeat(d.astype(np.float64), 32, axis=-1)


def rotate(x, pos, rot_dims, base, pairs):
    """x [n, heads, dim] fp32 at positions pos [n] -> fp64"""
    y = np.asarray(x, dtype=np.float64).copy()
    for i in range(rot_dims // 2):
        a, b = (2 * i, 2 * i + 1) if pairs == "adjacent" else (i, i + rot_dims // 2)
        t = np.asarray(pos, dtype=np.float64) * base ** (-2.0 * i / rot_dims)
        c, s = np.cos(t)[:, None], np.sin(t)[:, None]
        u, v = y[..., a].copy(), y[..., b].copy()
        y[..., a], y[..., b] = u * c - v * s, u * s + v * c
    return y


def positions(token_start, lengths):
    """(sequence, position) of rows token_start[0] .. token_start[-1] - 1"""
    out = []
    for s, n in enumerate(lengths):
        a, b = int(token_start[s]), int(token_start[s + 1])
        out += [(s, int(n) - b + i) for i in range(a, b)]
    return out


class Pages:
    """K and V rows as fp64 [n_pages, heads, page, dim] of what the cache holds"""

    def __init__(self, n_pages, page, heads, dim, dtype, rot_dims=0, base=10000.0, pairs="adjacent"):
        self.page, self.dtype, self.rot = page, dtype, (rot_dims, base, pairs)
        self.k = np.zeros((n_pages, heads, page, dim))
        self.v = np.zeros((n_pages, heads, page, dim))

    def append(self, k, v, table, token_start, lengths, q=None):
        at = positions(token_start, lengths)
        first = int(token_start[0])
        rows = range(first, first + len(at))
        pos = [p for _, p in at]
        kr = held(rotate(k[first:first + len(at)], pos, *self.rot).astype(np.float32), self.dtype)
        vr = held(v[first:first + len(at)], self.dtype)
        for i, (s, p) in enumerate(at):
            if p >= 0:
                self.k[table[s, p // self.page], :, p % self.page] = kr[i]
                self.v[table[s, p // self.page], :, p % self.page] = vr[i]
        if q is None:
            return None
        out = np.asarray(q, dtype=np.float64).copy()
        turned = rotate(q[first:first + len(at)], pos, *self.rot)
        for i, (_, p) in zip(rows, at):
            if p >= 0:
                out[i] = turned[i - first]
        return out

    def rows(self, which, s, n, table):
        """the first n rows of sequence s, [heads, n, dim]"""
        pool = self.k if which == "k" else self.v
        p = np.arange(n)
        return pool[table[s, p // self.page], :, p % self.page].transpose(1, 0, 2)

    def attend(self, q, table, token_start, lengths, scale, window=0, sinks=0, given=None):
        """outputs fp64 (rows of nobody as in `given`); per output sum p |v|; per row the largest scale * sum |q k|, then the dims' sums of |v|"""
        q = np.asarray(q, dtype=np.float64)
        out = np.zeros_like(q) if given is None else np.asarray(given, dtype=np.float64).copy()
        mass, reach = np.zeros_like(q), np.zeros(q.shape[:2] + (1 + q.shape[2],))
        first = int(token_start[0])
        for i, (s, p) in enumerate(positions(token_start, lengths)):
            i += first
            if p < 0:
                out[i] = 0
                continue
            t = np.arange(p + 1)
            seen = t[(t > p - window) | (t < sinks)] if window else t
            pg, r = table[s, seen // self.page], seen % self.page
            for h in range(q.shape[1]):
                g = h // (q.shape[1] // self.k.shape[1])
                k, v = self.k[pg, g, r], self.v[pg, g, r]
                z = k @ q[i, h] * scale
                w = np.exp(z - z.max())
                w /= w.sum()
                out[i, h] = w @ v
                mass[i, h] = w @ np.abs(v)
                reach[i, h, 0] = abs(scale) * (np.abs(k) @ np.abs(q[i, h])).max()
                reach[i, h, 1:] = np.abs(v).sum(axis=0)
        return out, mass, reach
