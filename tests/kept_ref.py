# SPDX-License-Identifier: Unlicense
"""Norms with codes, the cache of 8-bit keys and values and attention within a
window (include/ops.h) from their definitions, in numpy: roundings where the
definition has them, 64 bits otherwise."""

import numpy as np

import long_ref as ref
from long_ref import U


def rms_norm(x, r, g, eps):
    """(h, y) in float32, as the definition rounds them."""
    with np.errstate(all="ignore"):
        h = x if r is None else x + r
        inv = (1 / np.sqrt((h.astype(np.float64) ** 2).mean(-1, keepdims=True) + np.float64(np.float32(eps)))).astype(np.float32)
        y = h * inv
        return h, y if g is None else y * g


def pitch(d):
    return -(-d // 16) * 16


class Kept:
    """A cache: codes (pages, heads, page, pitch), scales (pages, heads, page)."""

    def __init__(self, pages, page, kv, d, seed=0):
        rng = np.random.default_rng(seed)
        self.pages, self.page, self.kv, self.d = pages, page, kv, d
        shape = (pages, kv, page, pitch(d))
        # What is there before: any bytes, with zeros behind the channels.
        self.kc, self.vc = (rng.integers(-127, 128, shape).astype(np.int8) for _ in "kv")
        self.kc[..., d:] = self.vc[..., d:] = 0
        self.ks, self.vs = (np.exp(rng.normal(-5, 0.5, shape[:3])).astype(np.float32) for _ in "kv")

    def places(self, start, length, table, rows):
        """(row, sequence, position, page or -1) of every row of a sequence."""
        for b in range(len(length)):
            s, e = (min(max(int(v), 0), rows) for v in start[b:b + 2])
            for row in range(s, e):
                p = max(int(length[b]), 0) - (e - row)
                page = int(table[b, p // self.page]) if 0 <= p < table.shape[1] * self.page else -1
                yield row, b, p, page if 0 <= page < self.pages else -1

    def write(self, k, v, start, length, table):
        for x, codes, scales in ((k, self.kc, self.ks), (v, self.vc, self.vs)):
            c, s = ref.quant(x)
            for row, _, p, page in self.places(start, length, table, len(k)):
                if page >= 0:
                    codes[page, :, p % self.page, :self.d] = c[row]
                    scales[page, :, p % self.page] = s[row]

    def read(self, start, length, table, k, v):
        """Into k, v (rows, heads, d): rows of no sequence stay."""
        for row, _, p, page in self.places(start, length, table, len(k)):
            for x, codes, scales in ((k, self.kc, self.ks), (v, self.vc, self.vs)):
                at = p % self.page
                x[row] = 0 if page < 0 else codes[page, :, at, :self.d].astype(np.float32) * scales[page, :, at][:, None]

    def keys(self, b, length, table):
        """Keys and values (n, heads, d) in 64 bits of sequence b, and which
        of them are kept."""
        n = min(max(int(length[b]), 0), table.shape[1] * self.page)
        pos = np.arange(n)
        page = table[b][pos // self.page] if n else np.zeros(0, int)
        kept = (page >= 0) & (page < self.pages)
        page = np.where(kept, page, 0)
        out = []
        for codes, scales in ((self.kc, self.ks), (self.vc, self.vs)):
            out.append(codes[page, :, pos % self.page, :self.d].astype(np.float64) *
                       scales[page, :, pos % self.page][..., None].astype(np.float64))
        return out[0], out[1], kept


def sees(p, n, left, right, sinks):
    """(queries, keys): which of n keys the positions p see."""
    p, j = np.asarray(p)[:, None], np.arange(n)[None]
    see = (j <= p + right) if right >= 0 else np.ones((len(p), n), bool)
    if left >= 0:
        see &= (j >= p - left) | (j < sinks)
    return see


def attend(q, k, v, see, scale):
    """q (n, heads, d) over k, v (keys, key heads, d) in 64 bits where see (n,
    keys): (out, bound), the bound on what float32 may be off. A score of d
    products, each rounded onto a sum and then scaled, is off by at most (d +
    8) U of its products' magnitudes `size`, its exponent's argument (twice
    that at most) by 4 more, and a weight's exponential by 4 U; a weight and
    the sum that divides it may both be off. n weights are added, and n
    products of weights and values, with a rounding each, of splits and their
    joining 64 more."""
    n, h, d = q.shape
    g = h // k.shape[1]
    out, bound = np.zeros((n, h, d)), np.zeros((n, h, d))
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    for i in range(h):
        for a in range(n):
            rows = np.flatnonzero(see[a])
            if not len(rows):
                continue
            s = scale * (k[rows, i // g] @ q[a, i])
            size = (abs(scale) * (np.abs(k[rows, i // g]) @ np.abs(q[a, i]))).max()
            p = np.exp(s - s.max())
            p /= p.sum()
            out[a, i] = p @ v[rows, i // g]
            bound[a, i] = U * (2 * ((d + 12) * size + 4) + 2 * len(rows) + 64) * (p @ np.abs(v[rows, i // g]))
    return out, bound
