# SPDX-License-Identifier: Unlicense
"""GPU: attention within a window where its kernels change hands (many rows and
few, keys in one part and in hundreds, every width and page), with values far
apart, on codes past 2^31 bytes, and replayed from graphs."""

import numpy as np
import pytest

import kept_ref
from kept_ref import sees
from test_cache_gpu import Held, pages_of
from test_window_gpu import check, data, run

pytestmark = pytest.mark.gpu


def some(rng, n, most=40):
    """Rows to look at: the ends, those around tiles' ends, others."""
    rows = {0, n - 1, *(i for i in (127, 128, 255, 256) if i < n), *rng.integers(0, n, most).tolist()}
    return np.array(sorted(rows))


# Queries, keys, heads, key heads, channels, left, right, first keys: tiles of
# 256 and of 128 rows, in one part and in several, joined by a wave and by four.
WIDE = [(8400, 8400, 8, 8, 32, 20, 20, 3), (8300, 8300, 8, 8, 20, 30, 0, 0), (8300, 8300, 8, 8, 7, 10, 10, 1),
        (4300, 4300, 8, 8, 64, 40, 40, 0), (4300, 4300, 8, 8, 36, 70, 0, 70), (4300, 4300, 8, 8, 61, 9, 9, 2),
        (300, 9000, 2, 1, 32, 4000, 0, 5), (300, 9000, 2, 1, 64, -1, 0, 0), (90, 12000, 3, 1, 128, -1, -1, 0),
        (90, 12000, 3, 1, 127, 6000, 100, 9), (400, 3000, 1, 1, 100, 2000, 0, 0), (40, 30000, 1, 1, 12, -1, -1, 0),
        (1, 30000, 1, 1, 32, -1, 0, 0), (2, 30000, 2, 2, 61, 25000, 0, 4), (16, 20000, 1, 1, 128, -1, -1, 0)]


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("nq,nk,h,kv,d,left,right,sinks", WIDE)
def test_wide(nq, nk, h, kv, d, left, right, sinks, masked, dev, ic):
    print(f"[window] {nq} x {nk}, {h}/{kv} x {d}: {left} {right} {sinks} {masked}", flush=True)
    rng = np.random.default_rng(nq + nk + d)
    q, k, v = data(nq, nk, h, kv, d)
    q0, scale = nk - nq, np.float32(d ** -0.5)
    mask = (rng.random(nk) < 0.7).astype(np.uint8) if masked else None
    if masked:
        mask[nk // 2:nk // 2 + 300] = 0
        k[mask == 0], v[mask == 0] = np.nan, np.inf
    got = run(dev, ic, q, k, v, q0, left, right, sinks, scale, mask)
    assert np.isfinite(got).all()
    rows = some(rng, nq, 12 if nk > 10000 else 40)
    see = sees(rows + q0, nk, left, right, sinks)
    if masked:
        see &= mask != 0
        k[mask == 0] = v[mask == 0] = 0
    check(got[rows], q[rows], k, v, see, scale)


# Key heads, heads, channels, page, lengths, new rows, left, first keys.
KEPT = [(8, 8, 64, 16, [4200], [4200], 50, 0), (8, 8, 32, 32, [8300, 10], [8300, 10], 20, 5), (8, 8, 128, 128, [4200], [4200], 40, 0),
        (8, 8, 100, 64, [4300, 3], [4200, 1], -1, 0), (1, 2, 64, 16, [9000], [300], -1, 0), (1, 2, 24, 128, [9000], [300], 5000, 7),
        (1, 3, 128, 64, [12000, 40], [90, 40], -1, 0), (2, 2, 128, 16, [30000], [1], -1, 0), (1, 1, 32, 32, [30000, 100], [1, 1], -1, 0),
        (1, 16, 64, 128, [20000], [1], 15000, 100), (2, 4, 112, 16, [50] * 130, [1] * 130, -1, 0), (1, 1, 40, 16, [33] * 70, [3] * 70, 8, 2)]


def call(dev, ic, held, s, rows, Q, O, h, left, sinks, scale, work):
    w = h * held.ref.d
    dev.api.ops_attention_cache(dev.po, held.p, ic.C.byref(s), rows, ic.mat(Q, 0, w), ic.mat(O, 0, w), h, left, sinks, scale,
                                work.mem)


def look(got, q, held, start, lengths, table, left, sinks, scale, rng, most=12):
    """Some rows of every fifth sequence, if there are many."""
    step = 1 if len(lengths) < 10 else 5
    for b in range(0, len(lengths), step):
        n, m = lengths[b], start[b + 1] - start[b]
        k, v, kept = held.ref.keys(b, lengths, table)
        rows = some(rng, m, most)
        see = sees(rows + n - m, len(k), left, 0, sinks) & kept
        check(got[start[b] + rows], q[start[b] + rows], k, v, see, scale)


@pytest.mark.parametrize("kv,h,d,page,lengths,new,left,sinks", KEPT)
def test_wide_cache(kv, h, d, page, lengths, new, left, sinks, dev, ic):
    print(f"[window] cache {h}/{kv} x {d}, pages of {page}, {lengths[:3]} {new[:3]}: {left} {sinks}", flush=True)
    rng = np.random.default_rng(h * 131 + d)
    pages = sum(-(-n // page) for n in lengths) + 3
    held, table = Held(dev, ic, pages, page, kv, d), pages_of(rng, lengths, page, pages, 2)
    start, rows = np.concatenate([[0], np.cumsum(new)]), sum(new)
    q = 1.5 * rng.standard_normal((rows, h, d)).astype(np.float32)
    Q, O, s = dev.upload(q), dev.zeros(rows * h * d), held.seqs(start, lengths, table)
    work = dev.alloc(dev.api.ops_attention_cache_work_bytes(rows, h, d))
    scale = np.float32(d ** -0.5)
    call(dev, ic, held, s, rows, Q, O, h, left, sinks, scale, work)
    look(dev.read(O).reshape(q.shape), q, held, start, lengths, table, left, sinks, scale, rng)


# Magnitudes of the values of key i (of n), a power of two each.
SPREADS = {
    "two levels": lambda rng, n: rng.choice([0, 25], n), "steps of 2^10": lambda rng, n: np.arange(n) * 40 // n - 20,
    "falling": lambda rng, n: 20 - np.arange(n) * 40 // n, "one large": lambda rng, n: 22 * (np.arange(n) == n // 3),
    "one small": lambda rng, n: -24 * (np.arange(n) == n // 3), "any": lambda rng, n: rng.integers(-60, 60, n),
    "within": lambda rng, n: rng.integers(-10, 1, n), "jump": lambda rng, n: 70 * (np.arange(n) > n // 2),
    "tiny": lambda rng, n: np.full(n, -120) + rng.integers(0, 5, n), "first ones": lambda rng, n: 18 * (np.arange(n) < 70),
}


def check_apart(got, q, k, v, see, scale):
    """To the bound of kept_ref.attend and what weights in two f16 parts add:
    a weight of 2^-25 steps where the largest value's is 2^10 or more is off by
    2^-35 of that value V, a key. Where all values that are kept lie within
    2^-12 of V that is all; where some are smaller or zero, rows whose largest
    output is under 2^-14 V are computed in float32, so that it is also no more
    than 2^-21 of the row's largest output, 2^-20 as that is itself off. Without it the first run was 873 times the bound
    off, in channels of 10^-22 beside others of 10^-2, from a cache's code of 0
    under nearly all of the weight."""
    want, bound = kept_ref.attend(q, k, v, see, scale)
    rows = np.abs(v).max(-1)
    largest = rows.max(0).repeat(q.shape[1] // k.shape[1])
    apart = (rows < 2.0 ** -12 * rows.max(0)).any(0).repeat(q.shape[1] // k.shape[1])
    own = 2.0 ** 15 * np.abs(want).max(-1)
    more = see.sum(1)[:, None] * 2.0 ** -35 * np.where(apart, np.minimum(largest, own), largest)
    err = np.abs(got - want)
    print(f"  worst {np.max(err / (bound + more[..., None] + 1e-37)):.3f} of the bound", flush=True)
    assert np.all(err <= bound + more[..., None] + 1e-37)


@pytest.mark.parametrize("spread", SPREADS)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("nq", [2, 150])
def test_values_apart(nq, d, spread, dev, ic):
    """Values of unlike magnitude, even weights and ones that part far, keys of
    no value: each output to the bound on its own terms, of float32 keys and of
    a cache."""
    nk, h, kv, page = 320, 2, 1, 64
    rng = np.random.default_rng(nq + d)
    q, k, v = data(nq, nk, h, kv, d)
    q *= np.exp(rng.normal(0, 1.5, (nq, h, 1))).astype(np.float32)
    v = (v * 2.0 ** SPREADS[spread](rng, nk)[:, None, None].astype(np.float64)).astype(np.float32)
    v[nk // 5::50] = 0
    scale, q0 = np.float32(d ** -0.5), nk - nq
    for left, sinks in ((-1, 0), (80, 3)):
        see = sees(np.arange(nq) + q0, nk, left, 0, sinks)
        check_apart(run(dev, ic, q, k, v, q0, left, 0, sinks, scale), q, k, v, see, scale)
    held = Held(dev, ic, nk // page, page, kv, d)
    table = np.arange(nk // page, dtype=np.int32)[None]
    s = held.seqs([0, nk], [nk], table)
    K, V = dev.upload(k), dev.upload(v)
    dev.api.ops_cache_write(dev.po, held.p, ic.C.byref(s), nk, ic.mat(K, 0, kv * d), ic.mat(V, 0, kv * d))
    held.ref.write(k, v, [0, nk], [nk], table)
    k8, v8, _ = held.ref.keys(0, [nk], table)
    t, Q, O = held.seqs([0, nq], [nk], table), dev.upload(q), dev.zeros(q.size)
    work = dev.alloc(dev.api.ops_attention_cache_work_bytes(nq, h, d))
    for left, sinks in ((-1, 0), (80, 3)):
        call(dev, ic, held, t, nq, Q, O, h, left, sinks, scale, work)
        check_apart(dev.read(O).reshape(q.shape), q, k8, v8, sees(np.arange(nq) + q0, nk, left, 0, sinks), scale)


@pytest.mark.parametrize("nq", [1, 200])
def test_a_key_without_value_wins(nq, dev, ic):
    """The first key takes nearly all weight and has values of zero or far
    smaller ones: what the others add stays."""
    nk, h, d = 256, 1, 64
    q, k, v = data(nq, nk, h, 1, d)
    q[..., 0] = 8
    k[..., 0] = 0
    for score, small in ((20, 0.0), (26, 0.0), (14, 2.0 ** -20), (18, 2.0 ** -25), (24, 2.0 ** -40)):
        k[0] = 0
        k[0, 0, 0] = score * d ** 0.5 / 8
        v2 = v.copy()
        v2[0] *= small
        see = sees(np.arange(nq) + nk - nq, nk, -1, -1, 0)
        check_apart(run(dev, ic, q, k, v2, nk - nq, -1, -1, 0, np.float32(d ** -0.5)), q, k, v2, see, np.float32(d ** -0.5))


def test_codes_past_2_to_31(dev, ic):
    """Pages whose codes start past byte 2^31, single tokens and a prompt."""
    kv, h, d, page, pages, n = 8, 16, 128, 128, 17000, 700
    if (pages - 8) * kv * page * d < 1 << 31:
        pytest.fail("pages end before 2^31")
    rng = np.random.default_rng(3)
    bufs = [dev.alloc(pages * kv * page * x) for x in (d, d, 4, 4)]
    cache = ic.Cache(*(b.mem for b in bufs), pages, page, kv, d)
    table = (pages - 1 - rng.permutation(8)[:6]).astype(np.int32)[None]
    k, v = (rng.standard_normal((n, kv, d)).astype(np.float32) for _ in "kv")
    ref = kept_ref.Kept(8, page, kv, d)
    ref.write(k, v, [0, n], [n], table - (pages - 8))
    k8, v8, _ = ref.keys(0, [n], table - (pages - 8))
    K, V, T, L = dev.upload(k), dev.upload(v), dev.upload(table), dev.upload(np.array([n], np.int32))
    scale = np.float32(d ** -0.5)
    for m in (n, 1):
        S = dev.upload(np.array([0, m], np.int32))
        s = ic.Seqs(S.mem, L.mem, T.mem, 1, 6)
        if m == n:
            dev.api.ops_cache_write(dev.po, ic.C.byref(cache), ic.C.byref(s), n, ic.mat(K, 0, kv * d), ic.mat(V, 0, kv * d))
        q = 1.5 * rng.standard_normal((m, h, d)).astype(np.float32)
        Q, O = dev.upload(q), dev.zeros(q.size)
        work = dev.alloc(dev.api.ops_attention_cache_work_bytes(m, h, d))
        dev.api.ops_attention_cache(dev.po, ic.C.byref(cache), ic.C.byref(s), m, ic.mat(Q, 0, h * d), ic.mat(O, 0, h * d), h, -1,
                                    0, scale, work.mem)
        rows = some(rng, m, 6)
        check(dev.read(O).reshape(q.shape)[rows], q[rows], k8, v8, sees(rows + n - m, n, -1, 0, 0), scale)


def test_window_in_graphs(dev, ic):
    """Two recordings of other sizes, replayed in turn on new values beside
    eager calls of their own: each replay as the eager call to the bit."""
    shapes = [(1, 5000, 4, 1, 64, -1, 0), (200, 900, 4, 2, 128, 100, 5)]
    scale, held = 0.1, []
    for nq, nk, h, kv, d, left, sinks in shapes:
        bufs = [dev.alloc(4 * x) for x in (nq * h * d, nk * kv * d, nk * kv * d, nq * h * d, nq * h * d)]
        work = [dev.alloc(dev.api.ops_attention_window_work_bytes(nq, h, d)) for _ in "ab"]

        def attend(out, w, b=bufs, work=work, a=(nq, nk, h, kv, d, nk - nq, left, 0, sinks)):
            dev.api.ops_attention_window(dev.po, ic.mat(b[0], 0, a[2] * a[4]), ic.mat(b[1], 0, a[3] * a[4]), ic.mat(b[2], 0, a[3] * a[4]),
                                         ic.mat(b[out], 0, a[2] * a[4]), *a, scale, None, work[w].mem)
        dev.api.ocl_graph_begin(dev.pb)
        attend(3, 0)
        held.append((bufs, attend, dev.api.ocl_graph_end(dev.pb), (nq, nk, h, kv, d)))
    try:
        for seed in range(3):
            for bufs, attend, graph, size in held:
                for b, x in zip(bufs, data(*size, seed)):
                    dev.write(b, x)
            for _, _, graph, _ in held:
                dev.api.ocl_graph_launch(dev.pb, graph)
            for bufs, attend, _, _ in held:
                attend(4, 1)
            for bufs, *_ in held:
                got, want = dev.read(bufs[3]), dev.read(bufs[4])
                assert np.array_equal(got, want) and got.any()
            dev.finish()
    finally:
        for _, _, graph, _ in held:
            ic.lib().ocl_graph_free(graph)


def test_single_tokens_from_a_graph(dev, ic):
    """One recording of write and attention serves every step: lengths and
    pages are read from device memory, over a page's end and where a sequence
    starts again from its first token."""
    kv, h, d, page, n = 4, 8, 64, 16, 3
    rng = np.random.default_rng(5)
    held = Held(dev, ic, 40, page, kv, d)
    lengths = np.array([14, 100, 31], np.int32)
    table = rng.permutation(40)[:n * 10].reshape(n, 10).astype(np.int32)
    start = np.arange(n + 1)
    s = held.seqs(start, lengths, table)
    Q, K, V, O = (dev.zeros(n * x * d) for x in (h, kv, kv, h))
    work, scale = dev.alloc(dev.api.ops_attention_cache_work_bytes(n, h, d)), np.float32(0.125)
    dev.api.ocl_graph_begin(dev.pb)
    dev.api.ops_cache_write(dev.po, held.p, ic.C.byref(s), n, ic.mat(K, 0, kv * d), ic.mat(V, 0, kv * d))
    call(dev, ic, held, s, n, Q, O, h, 40, 2, scale, work)
    graph = dev.api.ocl_graph_end(dev.pb)
    try:
        for step in range(5):
            lengths = lengths + 1
            if step == 3:
                lengths[1] = 1
                table[2] = rng.permutation(table[2])
            q, k, v = (rng.standard_normal((n, x, d)).astype(np.float32) for x in (h, kv, kv))
            for b, x in zip((Q, K, V, s.bufs[1], s.bufs[2]), (q, k, v, lengths, table)):
                dev.write(b, x)
            dev.api.ocl_graph_launch(dev.pb, graph)
            held.ref.write(k, v, start, lengths, table)
            held.matches()
            got = dev.read(O).reshape(q.shape)
            for b in range(n):
                k8, v8, kept = held.ref.keys(b, lengths, table)
                see = sees([lengths[b] - 1], len(k8), 40, 0, 2) & kept
                check(got[b:b + 1], q[b:b + 1], k8, v8, see, scale)
            call(dev, ic, held, s, n, Q, O, h, 40, 2, scale, work)
            assert np.array_equal(dev.read(O).reshape(q.shape), got)
            dev.finish()
    finally:
        ic.lib().ocl_graph_free(graph)


@pytest.mark.parametrize("before,new", [(600, 1), (600, 200), (1, 40)])
def test_rows_before_the_first_sequence(before, new, dev, ic):
    """Rows before start[0] are left as they are, and the first sequence's are
    computed once, over their queries too."""
    kv, h, d, page, n = 2, 8, 32, 16, 300
    rng = np.random.default_rng(before + new)
    held = Held(dev, ic, 40, page, kv, d)
    table = rng.permutation(40)[:38].reshape(2, 19).astype(np.int32)
    start, lengths, rows = [before, before + new, before + new + 3], [n, 77], before + new + 5
    q, scale = 1.5 * rng.standard_normal((rows, h, d)).astype(np.float32), np.float32(d ** -0.5)
    Q, s = dev.upload(q), held.seqs(start, lengths, table)
    work = dev.alloc(dev.api.ops_attention_cache_work_bytes(rows, h, d))
    call(dev, ic, held, s, rows, Q, Q, h, -1, 0, scale, work)
    got = dev.read(Q).reshape(q.shape)
    assert np.array_equal(got[:before], q[:before]) and np.array_equal(got[start[2]:], q[start[2]:])
    look(got, q, held, start, lengths, table, -1, 0, scale, rng)


@pytest.mark.parametrize("n", [64, 65, 700, 4097, 5000])
@pytest.mark.parametrize("d", [16, 40, 128])
def test_many_sequences(n, d, dev, ic):
    """More sequences than are looked at together, some without rows: written,
    read back, attended to."""
    kv, h, page = 1, 2, 16
    rng = np.random.default_rng(n + d)
    new = rng.choice([0, 1, 1, 1, 3], n)
    new[[0, n - 1]] = rng.integers(0, 2, 2)
    lengths = (new + rng.integers(0, 20, n)).astype(np.int32)
    table = np.arange(3 * n, dtype=np.int32).reshape(n, 3)
    start, rows = np.concatenate([[0], np.cumsum(new)]) + 2, int(new.sum()) + 5
    held = Held(dev, ic, 3 * n, page, kv, d)
    s = held.seqs(start, lengths, table)
    k, v, q = (rng.standard_normal((rows, x, d)).astype(np.float32) for x in (kv, kv, h))
    K, V, Q = dev.upload(k), dev.upload(v), dev.upload(q)
    dev.api.ops_cache_write(dev.po, held.p, ic.C.byref(s), rows, ic.mat(K, 0, d), ic.mat(V, 0, d))
    held.ref.write(k, v, start, lengths, table)
    held.matches()
    want = [np.full((rows, kv, d), 5, np.float32) for _ in "kv"]
    out = [dev.upload(x) for x in want]
    held.ref.read(start, lengths, table, *want)
    dev.api.ops_cache_read(dev.po, held.p, ic.C.byref(s), rows, *(ic.mat(o, 0, d) for o in out))
    for o, x in zip(out, want):
        assert np.array_equal(dev.read(o).reshape(x.shape), x)
    work, scale = dev.alloc(dev.api.ops_attention_cache_work_bytes(rows, h, d)), np.float32(d ** -0.5)
    call(dev, ic, held, s, rows, Q, Q, h, -1, 0, scale, work)
    got = dev.read(Q).reshape(q.shape)
    assert np.array_equal(got[:2], q[:2]) and np.array_equal(got[start[-1]:], q[start[-1]:])
    for b in {0, 1, n - 2, n - 1, *(i for i in (63, 64, 65, 127, 128, 4095, 4096) if i < n), *rng.integers(0, n, 30).tolist()}:
        at = slice(start[b], start[b + 1])
        if new[b]:
            k8, v8, kept = held.ref.keys(b, lengths, table)
            check(got[at], q[at], k8, v8, sees(np.arange(lengths[b] - new[b], lengths[b]), len(k8), -1, 0, 0) & kept, scale)


@pytest.mark.parametrize("scale", [0.0, -0.3])
@pytest.mark.parametrize("nq", [2, 90])
def test_other_scales(nq, scale, dev, ic):
    q, k, v = data(nq, 200, 2, 1, 48)
    see = sees(np.arange(nq) + 200 - nq, 200, 70, 0, 1)
    check(run(dev, ic, q, k, v, 200 - nq, 70, 0, 1, scale), q, k, v, see, np.float32(scale))


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("nq", [1, 90])
def test_values_of_zero(nq, d, dev, ic):
    """Zeros come out as zeros, beside a tile of others too."""
    q, k, v = data(nq, 300, 2, 1, d)
    v[:] = 0
    for some in (False, True):
        if some:
            v[:20] = 1
        got = run(dev, ic, q, k, v, 300 - nq, 40, 0, 0, 0.1)
        assert not got.any()
        see = sees(np.arange(nq) + 300 - nq, 300, -1, 0, 0)
        check(run(dev, ic, q, k, v, 300 - nq, -1, 0, 0, 0.1), q, k, v, see, np.float32(0.1))
