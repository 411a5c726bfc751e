# SPDX-License-Identifier: Unlicense
"""GPU: attention within a window and over a cache where queries and keys lie
far from 1, by all of its kernels: a row's result does not depend on how many
rows a call has."""

import numpy as np
import pytest

from kept_ref import sees
from test_cache_gpu import Held
from test_window_edges_gpu import call, some
from test_window_gpu import check, run

pytestmark = pytest.mark.gpu


def far(nq, nk, h, kv, d, power, signs, seed=0):
    """Queries of 2^-power and keys of 2^power, products of the order of 1:
    all below zero, or of both signs."""
    rng = np.random.default_rng(nq + nk + d + power + seed)
    q, k = (rng.uniform(0.5, 1.5, (n, x, d)) for n, x in ((nq, h), (nk, kv)))
    if signs == "mixed":
        q, k = (x * rng.choice([-1, 1], x.shape) for x in (q, k))
    else:
        q = -q
    v = rng.standard_normal((nk, kv, d))
    return (q * 2.0 ** -power).astype(np.float32), (k * 2.0 ** power).astype(np.float32), v.astype(np.float32)


@pytest.mark.parametrize("signs", ["below", "mixed"])
@pytest.mark.parametrize("power", [-112, -60, 60, 90, 100, 104, 112, 120])
@pytest.mark.parametrize("d", [30, 32, 64, 128])
@pytest.mark.parametrize("nq", [1, 200])
def test_queries_and_keys_far_from_1(nq, d, power, signs, dev, ic):
    """A score is of the order of 1, whatever its operands are."""
    nk, h, kv, page = 320, 2, 1, 64
    scale, q0 = np.float32(8 / d), nk - nq
    q, k, v = far(nq, nk, h, kv, d, power, signs)
    for left in (-1, 70):
        see = sees(np.arange(nq) + q0, nk, left, 0, 0)
        check(run(dev, ic, q, k, v, q0, left, 0, 0, scale), q, k, v, see, scale)
    held = Held(dev, ic, nk // page, page, kv, d)
    table = np.arange(nk // page, dtype=np.int32)[None]
    s, K, V = held.seqs([0, nk], [nk], table), dev.upload(k), dev.upload(v)
    dev.api.ops_cache_write(dev.po, held.p, ic.C.byref(s), nk, ic.mat(K, 0, kv * d), ic.mat(V, 0, kv * d))
    held.ref.write(k, v, [0, nk], [nk], table)
    k8, v8, _ = held.ref.keys(0, [nk], table)
    t, Q, O = held.seqs([0, nq], [nk], table), dev.upload(q), dev.zeros(q.size)
    work = dev.alloc(dev.api.ops_attention_cache_work_bytes(nq, h, d))
    for left in (-1, 70):
        call(dev, ic, held, t, nq, Q, O, h, left, 0, scale, work)
        check(dev.read(O).reshape(q.shape), q, k8, v8, sees(np.arange(nq) + q0, nk, left, 0, 0), scale)


@pytest.mark.parametrize("power", [102, 112])
@pytest.mark.parametrize("h,d,n", [(8, 32, 8400), (8, 64, 4300), (2, 128, 3000)])
def test_many_rows_of_large_keys(h, d, n, power, dev, ic):
    rng = np.random.default_rng(n)
    scale, left = np.float32(8 / d), 60
    q, k, v = far(n, n, h, h, d, power, "below")
    rows = some(rng, n)
    got = run(dev, ic, q, k, v, 0, left, 0, 0, scale)
    check(got[rows], q[rows], k, v, sees(rows, n, left, 0, 0), scale)
