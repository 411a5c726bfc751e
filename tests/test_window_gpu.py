# SPDX-License-Identifier: Unlicense
"""GPU: attention within a window and over the first keys, of float32 keys and
of a cache, against softmax(scale Q K^T) V in 64 bits (kept_ref.attend says what
float32 may be off)."""

import numpy as np
import pytest

import kept_ref
from kept_ref import sees
from test_cache_gpu import Held, pages_of

pytestmark = pytest.mark.gpu


def run(dev, ic, q, k, v, q0, left, right, sinks, scale, mask=None, pads=(0, 0, 0, 0), in_place=False):
    nq, h, d = q.shape
    nk, kv, _ = k.shape
    widths = (h * d, kv * d, kv * d, h * d)
    bufs = []
    for x, w, pad in zip((q, k, v, np.full((nq, h, d), 7, np.float32)), widths, pads):
        wide = np.full((max(1, len(x)), w + pad), 7, np.float32)
        wide[:len(x), :w] = x.reshape(len(x), w)
        bufs.append(dev.upload(wide))
    if in_place:
        bufs[3] = bufs[0]
        pads = (pads[0], pads[1], pads[2], pads[0])
    M = dev.upload(mask) if mask is not None else None
    work = dev.alloc(dev.api.ops_attention_window_work_bytes(nq, h, d))
    dev.api.ops_attention_window(dev.po, *(ic.mat(b, 0, w + p) for b, w, p in zip(bufs, widths, pads)), nq, nk, h, kv, d,
                                 q0, left, right, sinks, scale, ic.mem(M), work.mem)
    got = dev.read(bufs[3]).reshape(-1, h * d + pads[3])
    assert np.all(got[:, h * d:] == 7)
    return got[:nq, :h * d].reshape(nq, h, d)


def data(nq, nk, h, kv, d, seed=0):
    rng = np.random.default_rng(nq * 31 + nk * 7 + h + d + seed)
    q, k, v = (rng.standard_normal((n, g, d)).astype(np.float32) for n, g in ((nq, h), (nk, kv), (nk, kv)))
    return 1.5 * q, k, v


def check(got, q, k, v, see, scale):
    want, bound = kept_ref.attend(q, k, v, see, scale)
    err = np.abs(got - want)
    print(f"  worst {np.max(err / (bound + 1e-37), initial=0):.3f} of the bound", flush=True)
    assert np.all(err <= bound + 1e-37)


# Queries, keys, heads, key heads, channels, position of query 0, left, right,
# first keys.
CASES = [
    (1, 1, 1, 1, 1, 0, 0, 0, 0), (1, 0, 2, 1, 8, 0, 3, 0, 1), (5, 5, 2, 2, 16, 0, -1, 0, 0), (5, 5, 2, 2, 16, 0, -1, -1, 0),
    (7, 40, 4, 2, 32, 33, 8, 0, 2), (33, 33, 3, 1, 17, 0, 4, 4, 1), (64, 64, 2, 2, 33, 0, 10, 10, 0),
    (65, 129, 4, 1, 64, 64, 31, 0, 5), (100, 100, 8, 8, 32, 0, 0, 0, 0), (100, 100, 1, 1, 65, 0, 0, 3, 70),
    (130, 300, 4, 4, 100, 170, 63, 0, 4), (130, 300, 16, 4, 128, 170, 64, 5, 33), (200, 200, 2, 1, 96, 0, 199, 0, 0),
    (1, 700, 16, 4, 128, 699, 511, 0, 4), (1, 5000, 4, 1, 64, 4999, -1, 0, 0), (2, 3000, 8, 8, 40, 2998, 1000, 0, 64),
    (3, 2000, 12, 4, 128, 900, 300, 300, 1), (300, 2000, 2, 2, 64, 800, 100, 50, 10),
    # Positions before the first key, behind the last, and a window behind it.
    (20, 30, 2, 1, 32, -10, 5, 2, 3), (20, 30, 2, 1, 32, 25, 5, 2, 3), (4, 30, 2, 1, 32, 100, 20, 0, 0),
    (4, 30, 2, 1, 32, 100, 20, 0, 7), (3, 64, 6, 2, 72, 2000000000, 2147483647, 2147483647, 2147483647),
    (40, 64, 1, 1, 128, -2000000000, 5, 2147483647, 4), (150, 150, 7, 7, 48, 0, 1, 1, 150),
]


@pytest.mark.parametrize("nq,nk,h,kv,d,q0,left,right,sinks", CASES)
def test_window(nq, nk, h, kv, d, q0, left, right, sinks, dev, ic):
    print(f"[window] {nq} x {nk}, {h}/{kv} x {d}, {q0}: {left} {right} {sinks}", flush=True)
    q, k, v = data(nq, nk, h, kv, d)
    see = sees(np.arange(nq, dtype=np.int64) + q0, nk, left, right, sinks)
    check(run(dev, ic, q, k, v, q0, left, right, sinks, d ** -0.5), q, k, v, see, np.float32(d ** -0.5))


@pytest.mark.parametrize("d", [5, 32, 64, 70, 128])
@pytest.mark.parametrize("nq", [1, 140])
def test_mask(d, nq, dev, ic):
    """Stretches without data, rows whose window keeps no key, rows of a
    stride, an output over the queries."""
    nk, h, kv = 400, 4, 2
    q, k, v = data(nq, nk, h, kv, d)
    q0, left, right, sinks = nk - nq - 30, 20, 20, 3
    mask = (np.arange(nk) % 70 < 20).astype(np.uint8)
    mask[:2] = 0
    mask[0] = 255
    see = sees(np.arange(nq) + q0, nk, left, right, sinks) & (mask != 0)
    scale = np.float32(d ** -0.5)
    for kw in ({}, {"pads": (1, 2, 3, 5)}, {"in_place": True}):
        check(run(dev, ic, q, k, v, q0, left, right, sinks, scale, mask, **kw), q, k, v, see, scale)
    got = run(dev, ic, q, k, v, q0, left, right, 0, scale, np.zeros(nk, np.uint8))
    assert not got.any()


@pytest.mark.parametrize("d", [16, 64, 128])
@pytest.mark.parametrize("nq", [1, 70])
def test_values(d, nq, dev, ic):
    """What unseen keys and values hold does not matter; a seen NaN makes the
    rows that see it NaN and no other; large and tiny values keep their bits."""
    nk, h, kv, left, sinks = 300, 2, 1, 40, 2
    q, k, v = data(nq, nk, h, kv, d)
    q0, scale = nk - nq, np.float32(d ** -0.5)
    see = sees(np.arange(nq) + q0, nk, left, 0, sinks)
    far = ~see.any(0)
    k[far], v[far] = np.nan, np.inf
    clean = run(dev, ic, q, k, v, q0, left, 0, sinks, scale)
    k2, v2 = k.copy(), v.copy()
    k2[far] = v2[far] = 0
    check(clean, q, k2, v2, see, scale)
    for at in (nk - 1, 0, nk - nq // 2 - 1):
        for x in (k, v):
            y = x.copy()
            y[at, 0, d // 2] = np.nan
            got = run(dev, ic, q, y if x is k else k, y if x is v else v, q0, left, 0, sinks, scale)
            assert np.array_equal(np.isnan(got).any((1, 2)), see[:, at])
            # Other rows: the same as without it, to the bound.
            rest = ~see[:, at]
            if rest.any():
                check(got[rest], q[rest], k2, v2, see[rest], scale)
    for scale_v, scale_k in ((2.0 ** 90, 1), (2.0 ** -120, 1), (1, 2.0 ** -60), (1, 2.0 ** 40)):
        kk, vv = k2 * np.float32(scale_k), v2 * np.float32(scale_v)
        s = np.float32(scale / scale_k)
        check(run(dev, ic, q, kk, vv, q0, left, 0, sinks, s), q, kk, vv, see, s)
    # Weights that part far: a key that wins, beside values 2^60 larger.
    k3 = k2.copy()
    k3[-1] = 40 * q[-1, :1]
    v3 = v2.copy()
    v3[:-1] *= np.float32(2.0 ** 60)
    check(run(dev, ic, q, k3, v3, q0, left, 0, sinks, scale), q, k3, v3, see, scale)
    # Scores of infinity below: a key that no weight is left for.
    k4 = k2.copy()
    k4[-3:] = -3e38 * np.sign(q[-1, :1])
    got = run(dev, ic, q[-1:], k4, v2, nk - 1, left, 0, sinks, scale)
    fine = see[-1:].copy()
    fine[:, -3:] = False
    if d >= 64:
        check(got[:, :1], q[-1:, :1], k4, v2, fine, scale)


# Key heads, heads, channels, page, lengths, new rows, left, first keys.
KEPT = [
    (1, 1, 1, 16, [1], [1], -1, 0), (2, 4, 16, 16, [5], [5], -1, 0), (1, 4, 33, 32, [40, 1, 33], [3, 1, 33], 9, 2),
    (4, 16, 128, 64, [700, 64, 65, 1], [1, 1, 1, 1], -1, 0), (4, 16, 128, 64, [700, 64, 65, 1], [1, 1, 1, 1], 100, 4),
    (2, 2, 64, 128, [300], [300], 50, 10), (8, 8, 40, 16, [100, 0, 7], [17, 0, 7], 30, 0), (2, 16, 100, 32, [333, 50], [4, 50], -1, 0),
    (1, 8, 64, 64, [5000], [1], -1, 0), (1, 8, 64, 64, [5000], [1], 2000, 70), (2, 2, 32, 16, [900, 20], [150, 20], 64, 1),
    (4, 4, 128, 64, [260, 130], [140, 129], -1, 0), (1, 12, 96, 32, [77] * 20, [1] * 20, 40, 5), (3, 6, 20, 16, [200], [33], 0, 16),
]


@pytest.mark.parametrize("kv,h,d,page,lengths,new,left,sinks", KEPT)
def test_cache(kv, h, d, page, lengths, new, left, sinks, dev, ic):
    print(f"[window] cache {h}/{kv} x {d}, pages of {page}, {lengths} {new}: {left} {sinks}", flush=True)
    rng = np.random.default_rng(h * 131 + d)
    pages = sum(-(-n // page) for n in lengths) + 3
    held, table = Held(dev, ic, pages, page, kv, d), pages_of(rng, lengths, page, pages, 2)
    if left >= 0:
        # Pages behind every row's window are given back.
        for b, (n, m) in enumerate(zip(lengths, new)):
            gone = [i for i in range(table.shape[1]) if (i + 1) * page <= n - m - left and i * page >= sinks]
            table[b, gone] = -1
    start, rows = np.concatenate([[0], np.cumsum(new)]), sum(new) + 3
    q = 1.5 * rng.standard_normal((rows, h, d)).astype(np.float32)
    Q, O, s = dev.upload(q), dev.upload(np.full((rows, h * d + 1), 7, np.float32)), held.seqs(start, lengths, table)
    work = dev.alloc(dev.api.ops_attention_cache_work_bytes(rows, h, d))
    scale = np.float32(d ** -0.5)
    dev.api.ops_attention_cache(dev.po, held.p, ic.C.byref(s), rows, ic.mat(Q, 0, h * d), ic.mat(O, 0, h * d + 1), h, left,
                                sinks, scale, work.mem)
    got = dev.read(O).reshape(rows, h * d + 1)
    assert np.all(got[:, h * d] == 7) and np.all(got[start[-1]:] == 7)
    got = got[:, :h * d].reshape(rows, h, d)
    for b, (n, m) in enumerate(zip(lengths, new)):
        k, v, kept = held.ref.keys(b, lengths, table)
        see = sees(np.arange(n - m, n), n, left, 0, sinks) & kept
        at = slice(start[b], start[b + 1])
        check(got[at], q[at], k, v, see, scale)
    # The same over the queries.
    dev.api.ops_attention_cache(dev.po, held.p, ic.C.byref(s), rows, ic.mat(Q, 0, h * d), ic.mat(Q, 0, h * d), h, left,
                                sinks, scale, work.mem)
    again = dev.read(Q, rows * h * d).reshape(rows, h, d)
    assert np.array_equal(again[:start[-1]], got[:start[-1]]) and np.array_equal(again[start[-1]:], q[start[-1]:])


@pytest.mark.parametrize("d", [24, 128])
def test_cache_without_places(d, dev, ic):
    """Queries before the first position, lengths behind the table, pages given
    back within the window, a table of no pages, scales of NaN."""
    kv, h, page, rows = 2, 4, 16, 60
    rng = np.random.default_rng(d)
    held = Held(dev, ic, 6, page, kv, d)
    table = np.array([[3, -1, 0], [5, 6, -2147483648], [1, 2147483647, 4], [2, 2, 2]], np.int32)
    start, length = [0, 20, 26, 36, 39], [44, 4, 50, -5]
    q = 1.5 * rng.standard_normal((rows, h, d)).astype(np.float32)
    held.ref.vs[3, 0, 2] = held.ref.ks[0, 1, 9] = np.nan
    for b, x in ((2, held.ref.ks), (3, held.ref.vs)):
        dev.write(held.bufs[b], x)
    scale = np.float32(d ** -0.5)
    for left, sinks in ((-1, 0), (12, 2)):
        O, s = dev.upload(np.full((rows, h, d), 7, np.float32)), held.seqs(start, length, table)
        work, Q = dev.alloc(dev.api.ops_attention_cache_work_bytes(rows, h, d)), dev.upload(q)
        dev.api.ops_attention_cache(dev.po, held.p, ic.C.byref(s), rows, ic.mat(Q, 0, h * d), ic.mat(O, 0, h * d), h, left,
                                    sinks, scale, work.mem)
        got = dev.read(O).reshape(rows, h, d)
        assert np.all(got[39:] == 7)
        for b in range(4):
            k, v, kept = held.ref.keys(b, length, table)
            m = start[b + 1] - start[b]
            p = np.arange(m) + max(length[b], 0) - m
            see = sees(p, len(k), left, 0, sinks) & kept
            for i in range(h):
                bad = np.isnan(k[:, i // 2]).any(1) | np.isnan(v[:, i // 2]).any(1)
                mine = got[start[b]:start[b + 1], i:i + 1]
                nan = (see & bad).any(1)
                assert np.array_equal(np.isnan(mine).any((1, 2)), nan)
                z = [np.where(bad[:, None, None], 0, x[:, i // 2:i // 2 + 1]) for x in (k, v)]
                if m and (~nan).any():
                    check(mine[~nan], q[start[b]:start[b + 1], i:i + 1][~nan], *z, see[~nan], scale)
    empty = ic.Seqs(s.start, s.len, None, 4, 0)
    dev.api.ops_attention_cache(dev.po, held.p, ic.C.byref(empty), rows, ic.mat(Q, 0, h * d), ic.mat(O, 0, h * d), h, -1, 0,
                                scale, work.mem)
    got = dev.read(O).reshape(rows, h, d)
    assert not got[:39].any() and np.all(got[39:] == 7)
