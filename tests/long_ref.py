# SPDX-License-Identifier: Unlicense
"""The operators for long token sequences (include/ops.h) from their
definitions, in numpy: roundings where the definition has them, 64 bits
otherwise."""

import numpy as np

U = 2.0 ** -24
TINY = 2.0 ** -100


def pitch(c):
    return -(-c // 64) * 64


def quant(x):
    """Codes (int8) and scales of the rows of x (float32)."""
    x = np.asarray(x, np.float32)
    with np.errstate(all="ignore"):
        a = np.abs(x).max(-1)
        bad = ~np.isfinite(x).all(-1)
        live = ~bad & (a >= TINY)
        r = np.where(live, np.float32(127) / np.where(live, a, 1), 0).astype(np.float32)
        c = np.where(live[..., None], np.rint(x * r[..., None]), 0).astype(np.int8)
        s = np.where(bad, np.nan, np.where(live, a / np.float32(127), 0)).astype(np.float32)
    return c, s


def act(y, kind, slope=0.0):
    from math import erf
    if kind == 1:
        return 0.5 * y * (1 + np.vectorize(erf)(y / 2 ** 0.5))
    if kind == 2:
        return np.maximum(y, 0)
    if kind == 3:
        return np.where(y >= 0, y, slope * y)
    if kind == 4:
        return 0.5 * y * (1 + np.tanh((2 / np.pi) ** 0.5 * (y + 0.044715 * y ** 3)))
    return y


def rope(x, pos, freq, rot, interleaved, mult=1.0, inverse=False):
    """x (rows, heads, d), pos (rows, axes) -> the same rotated, in 64 bits."""
    x = x.astype(np.float64)
    p = np.arange(rot // 2)
    a = pos[:, p % pos.shape[1]].astype(np.float64) * freq
    a = (-a if inverse else a)[:, None]
    i, j = (2 * p, 2 * p + 1) if interleaved else (p, p + rot // 2)
    y = x.copy()
    y[..., i] = mult * (x[..., i] * np.cos(a) - x[..., j] * np.sin(a))
    y[..., j] = mult * (x[..., i] * np.sin(a) + x[..., j] * np.cos(a))
    return y


def index(k, bs, mask=None):
    """k (Nk, kv heads, d) -> codes (blocks, kv heads, d), scales."""
    nk, kv, d = k.shape
    n = -(-nk // bs)
    mean, count = np.zeros((n, kv, d), np.float32), np.zeros(n, int)
    for b in range(n):
        rows = np.arange(b * bs, min(nk, (b + 1) * bs))
        rows = rows if mask is None else rows[mask[rows] != 0]
        count[b] = len(rows)
        if len(rows):
            mean[b] = (k[rows].astype(np.float64).sum(0) / len(rows)).astype(np.float32)
    c, s = quant(mean)
    s[count == 0] = -1
    return c, s


def select(q, kc, ks, top):
    """q (Nq, heads, d), kc (blocks, kv heads, d) -> (Nq, heads, top) int32."""
    nq, h, d = q.shape
    n, kv, _ = kc.shape
    qc, qs = quant(q)
    sel = np.full((nq, h, top), -1, np.int32)
    for i in range(h):
        j = i // (h // kv)
        dot = qc[:, i].astype(np.int64) @ kc[:, j].astype(np.int64).T
        s = ks[:, j] * dot.astype(np.float32)
        s[np.isnan(qs[:, i])] = np.nan
        order = np.where(np.isnan(s), np.inf, s)
        order = np.where(np.isnan(s), 1, 0) * 1.0, order
        live = ~(ks[:, j] < 0)
        for a in range(nq):
            at = np.lexsort((np.arange(n), -order[1][a], -order[0][a]))
            at = at[live[at]][:top]
            sel[a, i, :len(at)] = at
    return sel


def attend(q, k, v, sel, bs, scale, mask=None):
    """(out, bound): softmax over the listed blocks in 64 bits, and how far
    float32 may be off (see test_blocks_gpu.py)."""
    nq, h, d = q.shape
    nk, kv, _ = k.shape
    n = -(-nk // bs) if nk else 0
    out, bound = np.zeros((nq, h, d)), np.zeros((nq, h, d))
    q64, k64, v64 = (x.astype(np.float64) for x in (q, k, v))
    for i in range(h):
        j = i // (h // kv)
        for a in range(nq):
            blocks = sorted({int(b) for b in sel[a, i] if 0 <= b < n})
            rows = np.array([r for b in blocks for r in range(b * bs, min(nk, (b + 1) * bs))], int)
            if mask is not None:
                rows = rows[mask[rows] != 0]
            if not len(rows):
                continue
            s = scale * (k64[rows, j] @ q64[a, i])
            size = (abs(scale) * (np.abs(k64[rows, j]) @ np.abs(q64[a, i]))).max()
            p = np.exp(s - s.max())
            p /= p.sum()
            out[a, i] = p @ v64[rows, j]
            units = len(blocks) * max(1, bs // 64)
            rel = 2 * ((d / 4 + 20) * size + 4) + min(len(rows), 64) + units + 48
            bound[a, i] = U * rel * (p @ np.abs(v64[rows, j]))
    return out, bound
