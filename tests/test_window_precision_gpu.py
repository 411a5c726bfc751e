# SPDX-License-Identifier: Unlicense
"""GPU: attention within a window and over a cache against 64 bits, by the
root mean square of the errors: what kept_stats.limits allows, which operands
of 16 bits pass (test_window_precision.py)."""

import numpy as np
import pytest

import kept_stats
from kept_ref import sees
from test_cache_gpu import Held, pages_of
from test_window_edges_gpu import KEPT, WIDE, call, some
from test_window_gpu import data, run

pytestmark = pytest.mark.gpu

# Between the few rows of one kernel and the tiles of another.
ROWS = [(16, 900, 4, 4, 64, 300, 0, 4), (17, 900, 4, 4, 64, 300, 0, 4), (4, 900, 16, 4, 128, -1, 0, 0), (5, 900, 16, 4, 128, -1, 0, 0),
        (130, 130, 4, 4, 128, -1, 0, 0), (257, 600, 8, 1, 32, -1, -1, 0), (700, 700, 16, 2, 64, 200, 50, 3)]


def check(got, q, k, v, see, scale):
    want, limit = kept_stats.attend(q, k, v, see, scale), kept_stats.limits(q, k, v, see, scale)
    rms, most = kept_stats.worst(got, want, limit)
    print(f"  root mean square {rms:.3f} of the limit, at most {most:.2f}", flush=True)
    assert rms <= 1 and most <= 12


@pytest.mark.parametrize("nq,nk,h,kv,d,left,right,sinks", WIDE + ROWS)
def test_window(nq, nk, h, kv, d, left, right, sinks, dev, ic):
    print(f"[window] {nq} x {nk}, {h}/{kv} x {d}: {left} {right} {sinks}", flush=True)
    q, k, v = data(nq, nk, h, kv, d)
    q0, scale = nk - nq, np.float32(d ** -0.5)
    got = run(dev, ic, q, k, v, q0, left, right, sinks, scale)
    rows = some(np.random.default_rng(d), nq, 12 if nk > 10000 else 40)
    check(got[rows], q[rows], k, v, sees(rows + q0, nk, left, right, sinks), scale)


@pytest.mark.parametrize("kv,h,d,page,lengths,new,left,sinks", KEPT)
def test_cache(kv, h, d, page, lengths, new, left, sinks, dev, ic):
    print(f"[window] cache {h}/{kv} x {d}, pages of {page}, {lengths[:3]} {new[:3]}: {left} {sinks}", flush=True)
    rng = np.random.default_rng(h * 131 + d)
    pages = sum(-(-n // page) for n in lengths) + 3
    held, table = Held(dev, ic, pages, page, kv, d), pages_of(rng, lengths, page, pages, 2)
    start, rows = np.concatenate([[0], np.cumsum(new)]), sum(new)
    k, v = (rng.standard_normal((sum(lengths), kv, d)).astype(np.float32) for _ in "kv")
    whole = np.concatenate([[0], np.cumsum(lengths)])
    K, V, t = dev.upload(k), dev.upload(v), held.seqs(whole, lengths, table)
    dev.api.ops_cache_write(dev.po, held.p, ic.C.byref(t), len(k), ic.mat(K, 0, kv * d), ic.mat(V, 0, kv * d))
    held.ref.write(k, v, whole, lengths, table)
    q = 1.5 * rng.standard_normal((rows, h, d)).astype(np.float32)
    Q, O, s = dev.upload(q), dev.zeros(rows * h * d), held.seqs(start, lengths, table)
    work = dev.alloc(dev.api.ops_attention_cache_work_bytes(rows, h, d))
    scale = np.float32(d ** -0.5)
    call(dev, ic, held, s, rows, Q, O, h, left, sinks, scale, work)
    got = dev.read(O).reshape(q.shape)
    for b in range(0, len(lengths), 1 if len(lengths) < 10 else 20):
        k8, v8, kept = held.ref.keys(b, lengths, table)
        at = some(rng, new[b], 12)
        see = sees(at + lengths[b] - new[b], len(k8), left, 0, sinks) & kept
        check(got[start[b] + at], q[start[b] + at], k8, v8, see, scale)
