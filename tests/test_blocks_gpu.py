# SPDX-License-Identifier: Unlicense
"""GPU: attention over selected blocks of keys, its index and its selection,
against their definitions.

Index and selection are equal to the bit: the 64-bit sum of at most 128
float32 values of like size is exact, its quotient and the codes round as IEEE
has it, the codes' product is a whole number. Attention: a score of d products
loses at most U (d / 4 + 18) of scale sum |q k| (U = 2^-24; lanes of d / 4
products and their sum, or six bf16 products each and the groups of them) and
the query's scaling 2 U, which a probability has relatively, with 4 U for its
exponential; numerator and denominator both carry it. A unit's sum over at
most 64 keys adds U of each, the merge one a unit, the division, the parts and
their scales 48 U: long_ref.attend's bound, of sum p |v|. That worst case would
hide a lost part, so the rms error is bounded too: scores of rms 1.5 have
sqrt((d / 4 + 18) / 3) roundings of random sign, none of more than U of 8 / ln
2; a unit's sum sqrt(64) / 2, the merge and the rest 8: within (12 + sqrt(d / 4
+ 18)) U of the output's rms. (Small parts lost in one of the two products make
2^-19 or more.)"""

import numpy as np
import pytest

import long_ref as ref
from long_ref import U

pytestmark = pytest.mark.gpu


class Case:
    """Operands on the device, rows strided and offset as asked."""

    def __init__(self, dev, ic, q, k, v, bs, top, scale, mask=None, off=0, pad=0):
        self.dev, self.ic, self.bs, self.top, self.scale = dev, ic, bs, top, scale
        (self.nq, self.h, self.d), (self.nk, self.kv, _) = q.shape, k.shape
        self.off, self.lq, self.lk = off, self.h * self.d + pad, self.kv * self.d + pad
        self.Q, self.K, self.V = (self._up(x, l) for x, l in ((q, self.lq), (k, self.lk), (v, self.lk)))
        self.O = dev.upload(np.full(off + self.nq * self.lq + 4, 7.0, np.float32))
        self.mask = dev.upload(mask) if mask is not None else None
        self.n = dev.api.ops_key_blocks(self.nk, bs)
        p = ref.pitch(self.d)
        self.KC = dev.upload(np.full(max(1, self.n * self.kv * p), 99, np.int8))
        self.KS = dev.upload(np.full(max(1, self.n * self.kv), 99.0, np.float32))
        self.SEL = dev.upload(np.full(self.nq * self.h * top + 4, 99, np.int32))
        need = max(dev.api.ops_attention_blocks_work_bytes(self.nq, self.nk, self.h, self.kv, self.d, bs, top),
                   dev.api.ops_block_select_work_bytes(self.nq, self.h, self.n, top))
        # Whatever the work buffer holds before must not matter.
        self.work = dev.upload(np.full((need + 19) // 4, np.nan, np.float32))

    def _up(self, x, ld):
        rows = x.reshape(len(x), x.shape[1] * x.shape[2])
        host = np.full(self.off + len(rows) * ld + 4, 7.0, np.float32)
        host[self.off:self.off + len(rows) * ld].reshape(len(rows), ld)[:, :rows.shape[1]] = rows
        return self.dev.upload(host)

    def index(self, b0=0, nb=None):
        self.dev.api.ops_block_index(self.dev.po, self.ic.mat(self.K, self.off, self.lk), self.nk, self.kv, self.d,
                                     self.bs, self.ic.mem(self.mask), b0, self.n - b0 if nb is None else nb,
                                     self.KC.mem, self.KS.mem)

    def codes(self):
        p = ref.pitch(self.d)
        kc = self.dev.read(self.KC, self.n * self.kv * p, np.int8).reshape(self.n, self.kv, p)
        assert not kc[..., self.d:].any()
        return kc[..., :self.d], self.dev.read(self.KS, self.n * self.kv).reshape(self.n, self.kv)

    def select(self):
        self.dev.api.ops_block_select(self.dev.po, self.ic.mat(self.Q, self.off, self.lq), self.nq, self.h, self.kv,
                                      self.d, self.KC.mem, self.KS.mem, self.n, self.top, self.SEL.mem, self.work.mem)

    def sel(self):
        s = self.dev.read(self.SEL, dtype=np.int32)
        assert (s[self.nq * self.h * self.top:] == 99).all()
        return s[:self.nq * self.h * self.top].reshape(self.nq, self.h, self.top)

    def attend(self, O=None):
        ic = self.ic
        self.dev.api.ops_attention_blocks(
            self.dev.po, ic.mat(self.Q, self.off, self.lq), ic.mat(self.K, self.off, self.lk),
            ic.mat(self.V, self.off, self.lk), ic.mat(O or self.O, self.off, self.lq), self.nq, self.nk, self.h,
            self.kv, self.d, self.bs, self.top, self.SEL.mem, self.scale, ic.mem(self.mask), self.work.mem)

    def out(self, O=None):
        o = self.dev.read(O or self.O)
        rows = o[self.off:self.off + self.nq * self.lq].reshape(self.nq, self.lq)
        w = self.h * self.d
        assert (o[:self.off] == 7).all() and (rows[:, w:] == 7).all() and (o[self.off + self.nq * self.lq:] == 7).all()
        return rows[:, :w].reshape(self.nq, self.h, self.d)


def draw(nq, nk, h, kv, d, masked=0, seed=0):
    rng = np.random.default_rng(nq + 3 * nk + d + seed)
    q, k, v = (rng.standard_normal((n, w, d)).astype(np.float32) for n, w in ((nq, h), (nk, kv), (nk, kv)))
    if nk:
        # Blocks that differ.
        k += rng.standard_normal((nk // 16 + 1, kv, d)).astype(np.float32).repeat(16, 0)[:nk]
    mask = (rng.random(nk) < 0.7).astype(np.uint8) if masked else None
    if masked and nk > 200:
        mask[64:200] = 0  # whole blocks
    return q, k, v, mask


def check(c, q, k, v, mask, sel, got):
    want, bound = ref.attend(q, k, v, sel, c.bs, c.scale, mask)
    worst = np.max(np.abs(got - want) / (bound + 1e-37))
    norm = np.linalg.norm(want)
    rms = np.linalg.norm(got - want) / norm if norm else 0.0
    print(f"[blocks] worst {worst:.3f} of the bound, rms {rms:.2e}", flush=True)
    assert worst <= 1
    assert rms <= U * (12 + (c.d / 4 + 18) ** 0.5)


# Nq, Nk, heads, kv heads, d, block, top, mask, offset, pad
SHAPES = [
    (1, 1, 1, 1, 1, 16, 1, 0, 0, 0), (1, 1000, 16, 4, 128, 64, 16, 0, 0, 0), (2, 70, 2, 1, 5, 16, 3, 1, 1, 3),
    (1, 333, 4, 4, 64, 128, 2, 1, 0, 0), (3, 129, 3, 3, 33, 32, 64, 0, 0, 0), (31, 400, 4, 2, 100, 64, 5, 1, 4, 8),
    (40, 640, 8, 8, 32, 32, 4, 0, 0, 0), (5, 4097, 4, 1, 64, 16, 9, 1, 0, 0), (33, 64, 2, 2, 64, 64, 1, 0, 2, 2),
    (7, 260, 2, 2, 128, 128, 8, 1, 3, 1), (1, 40000, 2, 1, 32, 16, 33, 0, 0, 0),
    # Many queries for few blocks: lists of rows.
    (700, 300, 4, 4, 64, 64, 3, 0, 0, 0), (650, 333, 4, 2, 32, 32, 4, 1, 0, 0), (600, 100, 4, 1, 128, 64, 2, 1, 0, 4),
    (900, 270, 2, 2, 33, 16, 7, 0, 1, 1), (800, 500, 4, 2, 40, 128, 2, 1, 0, 0), (513, 257, 8, 8, 65, 64, 4, 0, 0, 0),
    (2100, 129, 4, 4, 16, 16, 9, 1, 0, 0), (520, 1024, 8, 1, 64, 32, 16, 0, 0, 0), (560, 210, 8, 4, 128, 128, 1, 0, 0, 0),
    (1200, 150, 4, 2, 32, 64, 3, 1, 0, 0), (1300, 200, 4, 4, 20, 64, 3, 0, 1, 2), (700, 120, 4, 4, 128, 32, 3, 1, 0, 0),
    (700, 120, 4, 2, 90, 32, 3, 0, 2, 0)]
MANY = [(1, 20000), (300, 3000), (3000, 40), (4100, 300), (2100, 128), (4100, 500), (130, 2000)]


def test_every_kernel_is_among_the_shapes(dev, ic):
    """The shapes below and those of the selection's own tests reach every
    selection, the units one by one and by lists, of every width."""
    lib, how, sel = ic.lib(), set(), set()
    for nq, nk, h, kv, d, bs, top, *_ in SHAPES:
        lists = lib.icoreg_blocks_choice(nq, nk, h, kv, d, bs, top)
        how.add((lists, min(128, 32 << max(0, (d - 1) // 32)), lists and min(bs, 64) > 32, lists and d in (32, 64, 128)))
        sel.add(lib.icoreg_select_choice(dev.po, nq, h, kv, -(-nk // bs), top))
    assert {(0, d, 0, 0) for d in (32, 64, 128)} <= how
    assert {(1, d, k, f) for d in (32, 64, 128) for k in (False, True) for f in (False, True)} <= how
    for rows, n in MANY:
        sel.add(lib.icoreg_select_choice(dev.po, rows, 2, 1, n, 16))
    assert sel == {0, 1, 2}


@pytest.mark.parametrize("shape", SHAPES, ids=[str(s) for s in SHAPES])
def test_edges(shape, dev, ic):
    nq, nk, h, kv, d, bs, top, masked, off, pad = shape
    print(f"[blocks] {shape}", flush=True)
    q, k, v, mask = draw(nq, nk, h, kv, d, masked)
    c = Case(dev, ic, q, k, v, bs, top, float(np.float32(1.2 / d ** 0.5)), mask, off, pad)
    c.index()
    kc, ks = c.codes()
    want_c, want_s = ref.index(k, bs, mask)
    assert np.array_equal(ks, want_s) and np.array_equal(kc, want_c)
    c.select()
    sel = c.sel()
    assert np.array_equal(sel, ref.select(q, kc, ks, top))
    c.attend()
    check(c, q, k, v, mask, sel, c.out())


def test_refreshed_index(dev, ic):
    """Only the blocks asked for are written."""
    print("[blocks] refresh", flush=True)
    q, k, v, _ = draw(1, 300, 1, 2, 48)
    c = Case(dev, ic, np.repeat(q, 2, 1), k, v, 32, 4, 0.2)
    c.index(9, 1)
    c.index(2, 3)
    c.index(0, 0)
    kc, ks = c.dev.read(c.KC, c.n * 2 * 64, np.int8).reshape(c.n, 2, 64), c.dev.read(c.KS, c.n * 2).reshape(c.n, 2)
    want_c, want_s = ref.index(k, 32)
    made = [2, 3, 4, 9]
    assert np.array_equal(ks[made], want_s[made]) and np.array_equal(kc[made, :, :48], want_c[made])
    rest = np.delete(np.arange(c.n), made)
    assert (ks[rest] == 99).all() and (kc[rest] == 99).all()


# Few queries, and enough for tiles of rows.
TIES = [(5, 5), (64, 8), (65, 32), (65, 64), (200, 16), (256, 17), (500, 9), (513, 16), (1100, 64), (1600, 3), (9000, 20)]


@pytest.mark.parametrize("n,top,nq", [t + (9,) for t in TIES] + [t + (2100,) for t in TIES if t[0] <= 513] +
                         [t + (2400,) for t in TIES if 128 < t[0] <= 512])
def test_selection_of_ties(n, top, nq, dev, ic):
    """Scores that repeat, zeros of both signs, scales of zero, blocks without
    keys and NaN scales: lower blocks first."""
    print(f"[blocks] ties {n} {top} {nq}", flush=True)
    rng = np.random.default_rng(n)
    kv, d, h = 2, 16, 4
    kc = rng.integers(-2, 3, (n, kv, d)).astype(np.int8)
    ks = rng.choice([0.5, 0.5, 1.0, 0.0, -1.0], (n, kv)).astype(np.float32)
    if n > 500:
        ks[rng.integers(0, n, 3), 0] = np.nan
    q = rng.integers(-1, 2, (nq, h, d)).astype(np.float32)
    q[:, :, 0] = 2
    if nq > 9:
        # Scores that differ, too, and rows that go their own way among them.
        q[:1500] = rng.standard_normal((1500, h, d))
        q[700:703, 1] = np.inf
    q[1] = 0
    q[2, 1, 3], q[3, 2, 0], q[4] = np.nan, -np.inf, 1e-38
    full = np.zeros((n, kv, 64), np.int8)
    full[..., :d] = kc
    Q, KC, KS = dev.upload(q), dev.upload(full), dev.upload(ks)
    SEL = dev.upload(np.full(nq * h * top, 99, np.int32))
    work = dev.alloc(dev.api.ops_block_select_work_bytes(nq, h, n, top))
    dev.api.ops_block_select(dev.po, ic.mat(Q, 0, h * d), nq, h, kv, d, KC.mem, KS.mem, n, top, SEL.mem, work.mem)
    got = dev.read(SEL, dtype=np.int32).reshape(nq, h, top)
    assert np.array_equal(got, ref.select(q, kc, ks, top))


@pytest.mark.parametrize("rows,n", MANY)
def test_selection_of_many(rows, n, dev, ic):
    print(f"[blocks] many {rows} {n}", flush=True)
    rng = np.random.default_rng(rows)
    d, top = 128, 16
    kc = rng.integers(-127, 128, (n, 1, d)).astype(np.int8)
    ks = rng.random((n, 1)).astype(np.float32)
    q = rng.standard_normal((rows, 2, d)).astype(np.float32)
    Q, KC, KS = dev.upload(q), dev.upload(kc), dev.upload(ks)
    SEL = dev.upload(np.full(rows * 2 * top, 99, np.int32))
    work = dev.alloc(dev.api.ops_block_select_work_bytes(rows, 2, n, top))
    dev.api.ops_block_select(dev.po, ic.mat(Q, 0, 2 * d), rows, 2, 1, d, KC.mem, KS.mem, n, top, SEL.mem, work.mem)
    assert np.array_equal(dev.read(SEL, dtype=np.int32).reshape(rows, 2, top), ref.select(q, kc, ks, top))


@pytest.mark.parametrize("top", [7, 16, 31])
@pytest.mark.parametrize("d", [60, 128])
@pytest.mark.parametrize("n", [50, 128, 255, 512])
def test_selection_by_tiles(n, d, top, dev, ic):
    """Rows for the matrix instructions at every width of them: scores that
    differ, that repeat, blocks without keys, a query that is not finite."""
    print(f"[blocks] tiles {n} {d} {top}", flush=True)
    rows = 2700 if n <= 128 else 4700
    assert ic.lib().icoreg_select_choice(dev.po, rows, 2, 1, n, top) == 2
    rng = np.random.default_rng(n + d + top)
    full = np.zeros((n, 1, 64 if d <= 64 else 128), np.int8)
    full[..., :d] = rng.integers(-127, 128, (n, 1, d))
    kc = full[..., :d]
    kc[n // 3:n // 2] = kc[n // 3]
    ks = rng.random((n, 1)).astype(np.float32)
    ks[n // 3:n // 2] = 2.0
    ks[rng.integers(0, n, 5)] = -1.0
    q = rng.standard_normal((rows, 2, d)).astype(np.float32)
    q[:64] = rng.integers(-1, 2, (64, 2, d))
    q[1000, 1, 3] = np.inf
    Q, KC, KS = dev.upload(q), dev.upload(full), dev.upload(ks)
    SEL = dev.upload(np.full(rows * 2 * top, 99, np.int32))
    dev.api.ops_block_select(dev.po, ic.mat(Q, 0, 2 * d), rows, 2, 1, d, KC.mem, KS.mem, n, top, SEL.mem, None)
    assert np.array_equal(dev.read(SEL, dtype=np.int32).reshape(rows, 2, top), ref.select(q, kc, ks, top))


# Few queries, and enough for lists.
@pytest.mark.parametrize("nq", [3, 900])
@pytest.mark.parametrize("bs,d", [(64, 64), (32, 128), (128, 32), (16, 100), (32, 64)])
def test_lists_that_a_caller_makes(nq, bs, d, dev, ic):
    """Entries that are no block are skipped, blocks listed twice count once,
    rows that list nothing or only left-out keys are zero."""
    print(f"[blocks] lists {nq} {bs} {d}", flush=True)
    nk, h, kv, top = 300, 4, 2, 7
    q, k, v, mask = draw(nq, nk, h, kv, d, 1)
    mask[:] = 1
    mask[bs:2 * bs] = 0
    rng = np.random.default_rng(nq)
    c = Case(dev, ic, q, k, v, bs, top, float(np.float32(d ** -0.5)), mask)
    sel = rng.integers(-2, c.n + 2, (nq, h, top)).astype(np.int32)
    sel[0] = -1
    sel[1, 0], sel[1, 1] = 1, c.n  # the block without keys; none
    sel[2, 0] = c.n - 1
    sel[2, 1] = [0, 2 ** 31 - 1, -2 ** 31, 0, 0, 1, 0]
    dev.write(c.SEL, sel)
    c.attend()
    got = c.out()
    assert not got[0].any() and not got[1, :2].any()
    check(c, q, k, v, mask, sel, got)


@pytest.mark.parametrize("nq,nk,h,kv,d,bs,top", [
    (70001, 32003, 2, 1, 16, 16, 1), (70001, 32003, 2, 1, 33, 64, 1), (2503, 700, 2, 2, 64, 64, 3),
    (2503, 700, 4, 2, 128, 64, 3), (2503, 700, 2, 1, 128, 32, 3), (1301, 700, 8, 2, 50, 128, 3)])
def test_crowded_lists(nq, nk, h, kv, d, bs, top, dev, ic):
    """Every row lists the first block and stretches of rows the same others:
    lists of all rows (more than 2^16 of a key head), of whole tiles of 64 rows
    and of next to none."""
    print(f"[blocks] crowded {nq} {nk} {h} {kv} {d} {bs} {top}", flush=True)
    assert ic.lib().icoreg_blocks_choice(nq, nk, h, kv, d, bs, top) == 1
    q, k, v, _ = draw(nq, nk, h, kv, d)
    rng = np.random.default_rng(nq)
    c = Case(dev, ic, q, k, v, bs, top, d ** -0.5)
    sel = rng.integers(0, c.n, (nq // 97 + 1, h, top)).astype(np.int32).repeat(97, 0)[:nq]
    sel[:, :, 0] = np.where(np.arange(nq) % 11 < 10, 0, c.n - 1)[:, None]
    dev.write(c.SEL, np.concatenate([sel.ravel(), np.full(4, 99, np.int32)]))
    c.attend()
    got = c.out()
    some = np.unique(np.concatenate([rng.integers(0, nq, 1200), np.arange(0, 70), np.arange(nq - 70, nq)]))
    check(c, q[some], k, v, None, sel[some], got[some])
    c.attend()
    assert np.array_equal(c.out(), got)


@pytest.mark.parametrize("nq", [2, 700])
def test_no_keys(nq, dev, ic):
    print(f"[blocks] no keys {nq}", flush=True)
    q, k, v, _ = draw(nq, 0, 4, 2, 32)
    c = Case(dev, ic, q, k, v, 32, 3, 0.2)
    assert c.n == 0
    c.index()
    c.select()
    assert (c.sel() == -1).all()
    c.attend()
    assert not c.out().any()


@pytest.mark.parametrize("nq", [4, 800])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_values_that_are_not_finite(nq, d, dev, ic):
    """In left-out keys and values they do not matter; kept ones give what
    float32 gives: an infinite value an infinite output, a NaN score a NaN row,
    a score of minus infinity no weight. The other heads keep their values."""
    print(f"[blocks] not finite {nq} {d}", flush=True)
    nk, h, bs, top = 160, 6, 32, 3
    q, k, v, _ = draw(nq, nk, h, h, d)
    mask = np.ones(nk, np.uint8)
    mask[[3, 40, 159]] = 0
    c = Case(dev, ic, q, k, v, bs, top, float(np.float32(d ** -0.5)), mask)
    sel = np.tile(np.array([4, 0, 1], np.int32), (nq, h, 1))
    dev.write(c.SEL, sel)
    c.attend()
    clean = c.out()
    check(c, q, k, v, mask, sel, clean)
    q2, k2, v2 = q.copy(), k.copy(), v.copy()
    k2[3, 0], v2[3, 0], k2[40, 0], v2[159, 0] = np.nan, np.nan, np.inf, -np.inf  # left out
    v2[5, 1, 3], v2[6, 1, 7] = np.inf, 3.3e38
    k2[50, 2, 0] = np.nan
    q2[1, 3, 1] = np.nan
    k2[7, 4] = 0
    k2[7, 4, 0] = np.inf  # scores of either infinity, by the query's sign
    c2 = Case(dev, ic, q2, k2, v2, bs, top, c.scale, mask)
    dev.write(c2.SEL, sel)
    c2.attend()
    got = c2.out()
    assert np.array_equal(got[:, 0], clean[:, 0]) and np.array_equal(got[:, 5], clean[:, 5])
    assert np.all(got[:, 1, 3] == np.inf)
    rows = np.r_[128:160, 0:64]
    rows = rows[mask[rows] != 0]
    s = c.scale * q[:, 1].astype(np.float64) @ k[rows, 1].astype(np.float64).T
    p = np.exp(s - s.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    assert np.allclose(got[:, 1, 7], p[:, list(rows).index(6)] * 3.3e38, rtol=1e-4)
    assert np.allclose(np.delete(got[:, 1], [3, 7], 1), np.delete(clean[:, 1], [3, 7], 1), rtol=0, atol=1e-5)
    assert np.isnan(got[:, 2]).all()
    assert np.isnan(got[1, 3]).all()
    keep = np.delete(np.arange(nq), 1)
    assert np.array_equal(got[keep, 3], clean[keep, 3])
    up = q[:, 4, 0] > 0
    assert np.isnan(got[up, 4]).all() and np.isfinite(got[~up, 4]).all()
    rows = rows[rows != 7]
    s = c.scale * q[:, 4].astype(np.float64) @ k[rows, 4].astype(np.float64).T
    p = np.exp(s - s.max(1, keepdims=True))
    want = (p / p.sum(1, keepdims=True)) @ v[rows, 4].astype(np.float64)
    assert np.allclose(got[~up, 4], want[~up], rtol=0, atol=1e-5)


@pytest.mark.parametrize("nq", [3, 2400])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_scores_far_from_zero(nq, d, dev, ic):
    """Every score near -2^120 or 2^100: each query takes its best key's
    values, of the blocks that it lists."""
    print(f"[blocks] far from zero {nq} {d}", flush=True)
    rng = np.random.default_rng(d)
    nk, h, bs = 100, 2, 32
    q, k, v = (rng.uniform(0.5, 2, (n, h, d)).astype(np.float32) for n in (nq, nk, nk))
    for sign, e in ((-1, 60), (1, 50)):
        kk = np.ldexp(sign * k, e)
        c = Case(dev, ic, np.ldexp(q, e), kk, v, bs, 2, 0.125)
        sel = np.tile(np.array([2, 3], np.int32), (nq, h, 1))
        dev.write(c.SEL, sel)
        c.attend()
        got = c.out()
        s = sign * np.einsum("qhd,khd->hqk", q.astype(np.float64), k[64:].astype(np.float64))
        best = s.argmax(-1) + 64
        for i in range(h):
            assert np.allclose(got[:, i], v[best[i], i], rtol=8 * U, atol=0)


@pytest.mark.parametrize("nq", [2, 640, 3000])
@pytest.mark.parametrize("eq,ek,ev", [(-116, 116, 0), (90, -90, 0), (0, 0, -116), (0, 0, 60)])
def test_powers_of_two(eq, ek, ev, nq, dev, ic):
    """Scaling queries against keys, or values, by powers of two changes no
    bit but the exponents. Values of 2^-116 times small probabilities are
    subnormal: each of at most 2 x 64 products and as many sums of them may
    lose 2^-150, together 2^-142, of outputs of at least 2^-116: less than U /
    4. That moves the roundings that follow, of a unit's sum, of the merge's and
    of the quotient, by one place (2 U) each at most."""
    print(f"[blocks] 2^{eq} 2^{ek} 2^{ev} {nq}", flush=True)
    rng = np.random.default_rng(nq)
    h, d, nk = 2, 64, 128
    q, k, v = ((rng.uniform(1, 8, (n, h, d)) * rng.choice([-1, 1], (n, h, d))).astype(np.float32)
               for n in (nq, nk, nk))
    sel = np.tile(np.array([1, 0], np.int32), (nq, h, 1))
    outs = []
    for a, b, e in ((0, 0, 0), (eq, ek, ev)):
        c = Case(dev, ic, np.ldexp(q, a), np.ldexp(k, b), np.ldexp(np.abs(v), e), 64, 2, 0.0125)
        dev.write(c.SEL, sel)
        c.attend()
        outs.append(c.out())
    if ev > -100 or nq == 3000:  # lists: values are scaled
        assert np.array_equal(outs[1], np.ldexp(outs[0], ev))
    else:
        assert np.all(np.abs(np.ldexp(outs[1].astype(np.float64), -ev) - outs[0]) <= 6 * U * np.abs(outs[0]))


@pytest.mark.parametrize("nq", [3, 1500])
def test_output_in_place_and_packed(nq, dev, ic):
    """The output over the queries, in the middle of packed rows."""
    print(f"[blocks] in place {nq}", flush=True)
    h, d, bs, top = 4, 32, 32, 2
    q, k, v, _ = draw(nq, nq, h, h, d)
    w = h * d
    packed = dev.upload(np.concatenate([x.reshape(nq, w) for x in (k, q, v)], 1))
    c = Case(dev, ic, q, k, v, bs, top, 0.25)
    c.index()
    c.select()
    c.attend()
    m = lambda o: ic.mat(packed, o, 3 * w)  # noqa: E731
    dev.api.ops_attention_blocks(dev.po, m(w), m(0), m(2 * w), m(w), nq, nq, h, h, d, bs, top, c.SEL.mem, 0.25, None,
                                 c.work.mem)
    got = dev.read(packed, nq * 3 * w).reshape(nq, 3, h, d)
    assert np.array_equal(got[:, 1], c.out())
    assert np.array_equal(got[:, 0], k) and np.array_equal(got[:, 2], v)


@pytest.mark.parametrize("nq", [1, 2500])
def test_long_cache_offsets(nq, dev, ic):
    """Keys and values whose rows lie past 2^31 floats."""
    print(f"[blocks] long offsets {nq}", flush=True)
    nk, d, h, bs, ld = 70000, 64, 2, 64, 32768
    floats = (nk - 1) * ld + h * d
    assert floats > 2 ** 31
    K = dev.alloc(4 * (floats + 4))
    step = 1 << 28
    for o in range(0, floats, step):
        dev.api.ocl_fill(dev.pb, K.mem, o, min(step, floats - o), 0.0)
    rng = np.random.default_rng(nq)
    tail = rng.standard_normal((200, 2 * h * d)).astype(np.float32)
    for i in range(200):
        dev.write(K, tail[i, :h * d] if i == 199 else tail[i], 4 * (nk - 200 + i) * ld)
    # Values beside the keys; the last row's would lie behind the buffer.
    nk -= 1
    k = tail[:199, :h * d].reshape(199, h, d)
    v = tail[:199, h * d:].reshape(199, h, d)
    q = rng.standard_normal((nq, h, d)).astype(np.float32)
    n, top = dev.api.ops_key_blocks(nk, bs), 2
    Q, O = dev.upload(q), dev.zeros(nq * h * d)
    KC, KS = dev.alloc(n * h * 64), dev.alloc(n * h * 4)
    SEL = dev.upload(np.tile(np.array([n - 1, n - 2], np.int32), (nq, h, 1)))
    work = dev.alloc(dev.api.ops_attention_blocks_work_bytes(nq, nk, h, h, d, bs, top))
    dev.api.ops_block_index(dev.po, ic.mat(K, 0, ld), nk, h, d, bs, None, n - 1, 1, KC.mem, KS.mem)
    dev.api.ops_attention_blocks(dev.po, ic.mat(Q, 0, h * d), ic.mat(K, 0, ld), ic.mat(K, h * d, ld),
                                 ic.mat(O, 0, h * d), nq, nk, h, h, d, bs, top, SEL.mem, 0.125, None, work.mem)
    first = (n - 2) * bs - (nk - 199)
    assert first >= 0
    c = Case(dev, ic, q, k[first:], v[first:], bs, top, 0.125)
    got = dev.read(O, nq * h * d).reshape(nq, h, d)
    check(c, q, k[first:], v[first:], None, np.tile(np.array([1, 0], np.int32), (nq, h, 1)), got)
    want_c, want_s = ref.index(k[first:], bs)
    assert np.array_equal(dev.read(KS, h, np.float32, (n - 1) * h * 4), want_s[1])


@pytest.mark.parametrize("nq", [1, 512])
def test_recorded_and_replayed(nq, dev, ic):
    """Two recorded graphs with work buffers of their own, replayed in turn on
    changing inputs between eager calls."""
    print(f"[blocks] graph {nq}", flush=True)
    h, kv, d, nk, bs, top = 4, 2, 64, 400, 32, 4
    cases, graphs = [], []
    try:
        for s in range(2):
            q, k, v, mask = draw(nq, nk, h, kv, d, 1, s)
            c = Case(dev, ic, q, k, v, bs, top, 0.125, mask)
            dev.api.ocl_graph_begin(dev.pb)
            c.index()
            c.select()
            c.attend()
            graphs.append(dev.api.ocl_graph_end(dev.pb))
            cases.append([c, q, k, v, mask])
        for t in range(3):
            for i, (c, q, k, v, mask) in enumerate(cases):
                q = draw(nq, nk, h, kv, d, 0, 10 + t + i)[0]
                dev.write(c.Q, q)
                cases[i][1] = q
            for g in graphs:
                dev.api.ocl_graph_launch(dev.pb, g)
            for c, q, k, v, mask in cases:
                sel, got = c.sel(), c.out()
                kc, ks = c.codes()
                assert np.array_equal(sel, ref.select(q, kc, ks, top))
                check(c, q, k, v, mask, sel, got)
                c.index()
                c.select()
                c.attend()
                assert np.array_equal(c.out(), got)
    finally:
        for g in graphs:
            ic.lib().ocl_graph_free(g)


def test_results_do_not_depend_on_the_other_queries(dev, ic):
    """A query's output in a long batch, bit for bit, in batches that share
    nothing with it but the keys (both of many queries)."""
    print("[blocks] other queries", flush=True)
    h, kv, d, nk, bs, top = 4, 2, 64, 300, 64, 2
    q, k, v, _ = draw(3000, nk, h, kv, d)
    outs = []
    for lo, hi in ((0, 3000), (1400, 3000), (0, 1501)):
        c = Case(dev, ic, q[lo:hi], k, v, bs, top, 0.125)
        c.index()
        c.select()
        c.attend()
        outs.append((lo, c.out()))
    for lo, o in outs[1:]:
        assert np.array_equal(o, outs[0][1][lo:lo + len(o)])


@pytest.mark.parametrize("top", [2, 9])
@pytest.mark.parametrize("apart", [False, True], ids=["one unit", "two units"])
@pytest.mark.parametrize("ev", [70, 88])
@pytest.mark.parametrize("nq,bs,d", [(5, 32, 64), (5, 64, 128), (5, 128, 20), (2600, 32, 64), (2600, 64, 32),
                                     (2600, 64, 100), (2600, 32, 128), (2600, 128, 64)])
def test_small_weights_of_large_values(nq, bs, d, ev, apart, top, dev, ic):
    """A key of weight 1 beside keys of weights 2^-121 .. 2^-124 whose values
    are 2^139 times as large: the output is the latter's, and keeps float32's
    accuracy, in one unit of keys and in two, for few queries and for many.

    One product of a score is not zero, and has few bits. So a score's error is
    the scaling's: the constant log2 e, its product with scale, that with the
    query, and two roundings of the sum of its parts, 5 U of the score, which a
    weight has relatively beside 4 U for its exponential; the sums, the merge,
    the division and the parts as in long_ref.attend."""
    print(f"[blocks] small weights {nq} {bs} {d} 2^{ev} {apart} {top}", flush=True)
    h, nk = 2, 2 * bs
    rng = np.random.default_rng(nq + d + ev)
    assert ic.lib().icoreg_blocks_choice(nq, nk, h, h, d, bs, top) == (nq > 5)
    q, k, v = (rng.uniform(1, 2, (n, h, d)) for n in (nq, nk, nk))
    k[:], v[:] = 0, 0
    q[..., 0] = np.where(np.arange(nq) % 2, 255 / 256, 127 / 128)[:, None]
    small = np.arange(bs + 3, bs + 9) if apart else np.arange(3, 9)
    k[..., 0] = -2000.0
    k[0, :, 0] = 0
    k[small, :, 0] = -rng.integers(122, 125, (6, h))
    v[0] = np.ldexp(rng.uniform(-2, 2, (h, d)), ev - 139)
    v[small] = np.ldexp(rng.uniform(1, 2, (6, h, d)), ev)
    scale = float(np.float32(np.log(2)))
    q, k, v = (x.astype(np.float32) for x in (q, k, v))
    c = Case(dev, ic, q, k, v, bs, top, scale)
    sel = np.full((nq, h, top), -1, np.int32)
    sel[..., -2:] = [1, 0]
    dev.write(c.SEL, sel)
    c.attend()
    got = c.out().astype(np.float64)
    s = scale * np.einsum("qh,kh->qhk", q[..., 0].astype(np.float64), k[..., 0].astype(np.float64))
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    want = np.stack([p[:, i] @ v[:, i].astype(np.float64) for i in range(h)], 1)
    size = np.abs(s[..., np.r_[0, small]]).max()
    rel = 2 * (5 * size + 4) + 64 + 4 + 48
    # Values of one sign where they count: sum p |v| is the output.
    worst = np.max(np.abs(got - want) / (U * rel * want))
    print(f"[blocks] worst {worst:.3f} of the bound", flush=True)
    assert (want > 0).all() and worst <= 1


# Queries a pass at most, passes, lists; then Nq, Nk, heads, kv heads, d,
# block, top, mask, offset, pad. The last pass is shorter in all but the last.
PASSES = [
    (700, 2, 1, (1025, 300, 4, 4, 64, 64, 3, 1, 0, 0)), (700, 3, 1, (2000, 500, 6, 2, 33, 32, 4, 0, 2, 3)),
    (110, 3, 1, (299, 2000, 2, 1, 128, 128, 64, 1, 0, 0)), (600, 4, 1, (2399, 90, 3, 1, 32, 16, 6, 1, 1, 0)),
    (3, 3, 0, (7, 1000, 4, 2, 64, 16, 9, 1, 0, 4)), (9, 2, 0, (17, 3000, 6, 2, 100, 128, 11, 0, 1, 0)),
    (1, 5, 0, (5, 400, 2, 2, 32, 32, 2, 0, 0, 0))]


@pytest.mark.parametrize("place", ["apart", "over the queries"])
@pytest.mark.parametrize("most,passes,lists,shape", PASSES, ids=[str(p[3]) for p in PASSES])
def test_passes(most, passes, lists, shape, place, dev, ic):
    """Calls whose work is held to a few queries' are cut in passes: what one
    pass computes, bit for bit, and the definition; nothing behind the
    work that they say they use."""
    print(f"[blocks] passes {passes} {shape} {place}", flush=True)
    nq, nk, h, kv, d, bs, top, masked, off, pad = shape
    q, k, v, mask = draw(nq, nk, h, kv, d, masked)
    if masked:
        # A unit whose values go by float32.
        mask[nk // 2], v[nk // 2, 0] = 1, v[nk // 2, 0] * 2.0 ** 80
    scale, lib, used = float(np.float32(1.2 / d ** 0.5)), ic.lib(), ic.C.c_size_t()
    sizes, outs, sel = (nq, nk, h, kv, d, bs, top), [], None
    dp = 32 if d <= 32 else 64 if d <= 64 else 128
    query = h * top * max(1, bs // 64) * (dp + 2) * 4 + h * (-(-nk // bs)) // 8 + 1
    try:
        for budget, n in ((0, 1), (most * query, passes)):
            lib.icoreg_blocks_budget(budget)
            assert lib.icoreg_blocks_passes(*sizes, ic.C.byref(used)) == n
            assert lib.icoreg_blocks_choice(*sizes) == lists
            c = Case(dev, ic, q, k, v, bs, top, scale, mask, off, pad)
            if sel is None:
                c.index()
                c.select()
                sel = c.sel()
                # A row of nothing in every pass.
                sel[::97] = -1
            dev.write(c.SEL, sel)
            O = c.Q if place != "apart" else None
            c.attend(O)
            outs.append(c.out(O))
            assert used.value <= dev.api.ops_attention_blocks_work_bytes(*sizes)
            assert np.isnan(dev.read(c.work)[used.value // 4:]).all()
    finally:
        lib.icoreg_blocks_budget(0)
    assert np.array_equal(outs[0], outs[1])
    border = np.arange(-(-nq // passes), nq, -(-nq // passes))
    some = np.unique(np.clip(np.r_[0, nq - 1, 97, border - 1, border, border + 1,
                                   np.random.default_rng(nq).integers(0, nq, 60)], 0, nq - 1))
    check(c, q[some], k, v, mask, sel[some], outs[1][some])
    assert not outs[1][::97].any()


@pytest.mark.parametrize("place", ["apart", "over the queries"])
def test_passes_of_a_long_batch(place, dev, ic):
    """So many queries that the library cuts them by itself."""
    print(f"[blocks] long batch {place}", flush=True)
    nq, nk, h, kv, d, bs, top = sizes = (15901, 2000, 8, 2, 64, 64, 16)
    assert ic.lib().icoreg_blocks_passes(*sizes, None) == 2 and ic.lib().icoreg_blocks_choice(*sizes) == 1
    q, k, v, _ = draw(nq, nk, h, kv, d)
    c = Case(dev, ic, q, k, v, bs, top, 0.125)
    c.index()
    c.select()
    sel = c.sel()
    O = c.Q if place != "apart" else None
    c.attend(O)
    some = np.r_[0:3, 7948:7953, 15898:15901, np.random.default_rng(1).integers(0, nq, 40)]
    check(c, q[some], k, v, None, sel[some], c.out(O)[some])


@pytest.mark.parametrize("nq", [2, 130])
@pytest.mark.parametrize("d", [24, 64, 100])
def test_longest_lists(nq, d, dev, ic):
    """64 blocks of 128 keys a row, 128 units to merge: one by one and by lists."""
    print(f"[blocks] longest lists {nq} {d}", flush=True)
    nk, h, kv, bs, top = 9000, 2, 1, 128, 64
    assert ic.lib().icoreg_blocks_choice(nq, nk, h, kv, d, bs, top) == (nq > 2)
    q, k, v, mask = draw(nq, nk, h, kv, d, 1)
    c = Case(dev, ic, q, k, v, bs, top, float(np.float32(1.2 / d ** 0.5)), mask)
    c.index()
    c.select()
    sel = c.sel()
    kc, ks = c.codes()
    assert np.array_equal(sel, ref.select(q, kc, ks, top)) and (sel >= 0).all()
    c.attend()
    some = np.unique(np.r_[0, 1, nq - 1, np.random.default_rng(d).integers(0, nq, 12)])
    check(c, q[some], k, v, mask, sel[some], c.out()[some])
