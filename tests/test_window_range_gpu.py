# SPDX-License-Identifier: Unlicense
"""GPU: attention within a window and over a cache where queries and keys lie
far from 1, by all of its kernels: a row's result does not depend on how many
rows a call has."""

import numpy as np
import pytest

import kept_ref
from kept_ref import sees
from long_ref import U
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


def check_lost(got, q, k, v, see, scale):
    """To the bound of kept_ref.attend and what the channels far below a query's
    or key's largest may lose: 2^-20 of a score to base 2, so that a weight and
    the sum that divides it are off by 2^-20 ln 2 each, 22.2 units of 2^-24 together."""
    want, bound = kept_ref.attend(q, k, v, see, scale)
    bound += 23 * U * kept_ref.attend(q, k, np.abs(v), see, scale)[0]
    err = np.abs(got - want)
    print(f"  worst {np.max(err / (bound + 1e-37)):.3f} of the bound", flush=True)
    assert np.all(err <= bound + 1e-37)


@pytest.mark.parametrize("power", [4, 9, 14, 18, 20, 24, 30, 60, 100])
@pytest.mark.parametrize("d", [30, 32, 64, 128])
@pytest.mark.parametrize("nq", [2, 200])
def test_one_large_channel(nq, d, power, dev, ic):
    """A channel of the keys or of the queries far above the others, where the
    other side has nothing: the others' products are the scores."""
    nk, h, kv, page = 320, 2, 1, 64
    rng = np.random.default_rng(nq + d + power)
    scale, q0 = np.float32(2 * d ** -0.5), nk - nq
    q, k, v = (rng.standard_normal((n, x, d)).astype(np.float32) for n, x in ((nq, h), (nk, kv), (nk, kv)))
    many, zero = k.copy(), q.copy()
    many[::3, :, d // 2], zero[:, :, d // 2] = 2.0 ** power, 0
    few, large = k.copy(), q.copy()
    few[:, :, d // 2], large[::2, :, d // 2] = 0, 2.0 ** power
    for left in (-1, 70):
        see = sees(np.arange(nq) + q0, nk, left, 0, 0)
        for a, b in ((zero, many), (large, few)):
            check_lost(run(dev, ic, a, b, v, q0, left, 0, 0, scale), a, b, v, see, scale)
    held = Held(dev, ic, nk // page, page, kv, d)
    table = np.arange(nk // page, dtype=np.int32)[None]
    s, K, V = held.seqs([0, nk], [nk], table), dev.upload(few), dev.upload(v)
    dev.api.ops_cache_write(dev.po, held.p, ic.C.byref(s), nk, ic.mat(K, 0, kv * d), ic.mat(V, 0, kv * d))
    held.ref.write(few, v, [0, nk], [nk], table)
    k8, v8, _ = held.ref.keys(0, [nk], table)
    t, Q, O = held.seqs([0, nq], [nk], table), dev.upload(large), dev.zeros(q.size)
    work = dev.alloc(dev.api.ops_attention_cache_work_bytes(nq, h, d))
    for left in (-1, 70):
        call(dev, ic, held, t, nq, Q, O, h, left, 0, scale, work)
        check_lost(dev.read(O).reshape(q.shape), large, k8, v8, sees(np.arange(nq) + q0, nk, left, 0, 0), scale)


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("h,d,n", [(8, 32, 8400), (8, 64, 4300), (2, 128, 3000)])
def test_one_large_key(h, d, n, masked, dev, ic):
    """A key of one large channel among ordinary ones, and others that are left
    out and hold anything: rows that see it and rows that do not."""
    rng = np.random.default_rng(n)
    scale, left = np.float32(d ** -0.5), 60
    q, k, v = (rng.standard_normal((n, h, d)).astype(np.float32) for _ in "qkv")
    at = n // 2 + 5
    k[at, :, 0], q[:, :, 0] = 2.0 ** 28, 0
    mask = None
    if masked:
        mask = (rng.random(n) < 0.8).astype(np.uint8)
        mask[at] = 1
        k[mask == 0], v[mask == 0] = np.inf, np.nan
    rows = np.unique(np.concatenate([some(rng, n), np.arange(at - 3, at + left + 4)]))
    got = run(dev, ic, q, k, v, 0, left, 0, 0, scale, mask)
    see = sees(rows, n, left, 0, 0)
    if masked:
        see &= mask != 0
        k[mask == 0] = v[mask == 0] = 0
    check_lost(got[rows], q[rows], k, v, see, scale)


@pytest.mark.parametrize("power", [74, 76, 77, 78, 79, 80, 82, 100, 101, 102, 103, 104, 106, 108, 112])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("nq", [1, 2, 200])
def test_large_values(nq, d, power, dev, ic):
    """Sums of values below 2^115 do not pass float32's range on the way to an
    output."""
    nk, h, kv, page = 320, 2, 1, 64
    rng = np.random.default_rng(nq + d + power)
    scale, q0 = np.float32(d ** -0.5), nk - nq
    q, k = (rng.standard_normal((n, x, d)).astype(np.float32) for n, x in ((nq, h), (nk, kv)))
    v = (rng.uniform(1, 2, (nk, kv, d)) * np.where(np.arange(d) % 3 == 0, -1, 1) * 2.0 ** power).astype(np.float32)
    see = sees(np.arange(nq) + q0, nk, -1, 0, 0)
    check(run(dev, ic, q, k, v, q0, -1, 0, 0, scale), q, k, v, see, scale)
    held = Held(dev, ic, nk // page, page, kv, d)
    table = np.arange(nk // page, dtype=np.int32)[None]
    s, K, V = held.seqs([0, nk], [nk], table), dev.upload(k), dev.upload(v)
    dev.api.ops_cache_write(dev.po, held.p, ic.C.byref(s), nk, ic.mat(K, 0, kv * d), ic.mat(V, 0, kv * d))
    held.ref.write(k, v, [0, nk], [nk], table)
    k8, v8, _ = held.ref.keys(0, [nk], table)
    t, Q, O = held.seqs([0, nq], [nk], table), dev.upload(q), dev.zeros(q.size)
    work = dev.alloc(dev.api.ops_attention_cache_work_bytes(nq, h, d))
    call(dev, ic, held, t, nq, Q, O, h, -1, 0, scale, work)
    check(dev.read(O).reshape(q.shape), q, k8, v8, see, scale)


@pytest.mark.parametrize("power", [8, 14, 18, 22, 26, 40, 72])
@pytest.mark.parametrize("d", [12, 32, 50, 64, 128])
@pytest.mark.parametrize("nq", [2, 200])
def test_values_of_one_large_channel(nq, d, power, dev, ic):
    """A channel of all values, of some keys' or of one key's, far above the
    others. Few rows: each channel to the bound on its own terms. Many: to what
    two f16 parts add to it, a value 2^-39 of its row's largest (with its weight's
    parts 2^-38), a weight check_apart's share of the largest value."""
    nk, h, kv = 320, 2, 1
    rng = np.random.default_rng(nq + d + power)
    scale, q0 = np.float32(d ** -0.5), nk - nq
    q, k, v = (rng.standard_normal((n, x, d)).astype(np.float32) for n, x in ((nq, h), (nk, kv), (nk, kv)))
    for keys in (slice(None), slice(None, None, 7), slice(nk - 40, nk - 39)):
        w = v.copy()
        w[keys, :, d // 2] *= np.float32(2.0 ** power)
        for left in (-1, 70):
            see = sees(np.arange(nq) + q0, nk, left, 0, 0)
            want, bound = kept_ref.attend(q, k, w, see, scale)
            err = np.abs(run(dev, ic, q, k, w, q0, left, 0, 0, scale) - want)
            if nq > 16:
                rows = np.abs(w).max(-1).astype(np.float64)
                bound += 2.0 ** -38 * kept_ref.attend(q, k, np.repeat(rows[..., None], d, 2), see, scale)[0]
                own = np.minimum(rows.max(0), 2.0 ** 15 * np.abs(want).max(-1))
                bound += see.sum(1)[:, None, None] * 2.0 ** -35 * own[..., None]
            print(f"  worst {np.max(err / (bound + 1e-37)):.3f} of the bound", flush=True)
            assert np.all(err <= bound + 1e-37)
