# SPDX-License-Identifier: Unlicense
"""GPU: keys and values written to a cache's pages in 8 bits and read back,
against the definition, whose codes and scales are defined to the bit: no
tolerance, and every place that no row has as it was."""

import numpy as np
import pytest

from kept_ref import Kept

pytestmark = pytest.mark.gpu


class Held:
    """A cache on the device beside its numpy form."""

    def __init__(self, dev, ic, pages, page, kv, d, seed=0):
        self.dev, self.ic, self.ref = dev, ic, Kept(pages, page, kv, d, seed)
        self.bufs = [dev.upload(x) for x in (self.ref.kc, self.ref.vc, self.ref.ks, self.ref.vs)]
        self.struct = ic.Cache(*(b.mem for b in self.bufs), pages, page, kv, d)
        self.p = ic.C.pointer(self.struct)

    def seqs(self, start, length, table):
        table = np.ascontiguousarray(table, np.int32)
        bufs = [self.dev.upload(np.asarray(x, np.int32)) for x in (start, length)] + [self.dev.upload(table)]
        s = self.ic.Seqs(*(b.mem for b in bufs), len(length), table.shape[1])
        s.bufs = bufs
        return s

    def matches(self):
        for b, x in zip(self.bufs, (self.ref.kc, self.ref.vc, self.ref.ks, self.ref.vs)):
            got = self.dev.read(b, x.size, x.dtype).reshape(x.shape)
            assert np.array_equal(got, x, equal_nan=x.dtype == np.float32)


def pages_of(rng, lengths, page, pages, extra=0):
    """A table of distinct pages in no order for sequences of these lengths."""
    width = max(1, max(-(-n // page) for n in lengths)) + extra
    table = np.full((len(lengths), width), -1, np.int32)
    order = iter(rng.permutation(pages))
    for b, n in enumerate(lengths):
        for i in range(-(-n // page)):
            table[b, i] = next(order)
    return table


# Key heads, channels, page, lengths of the sequences, new rows of each.
CASES = [(1, 1, 16, [1], [1]), (2, 16, 16, [5], [5]), (3, 17, 32, [40, 1, 33], [3, 1, 33]),
         (4, 32, 64, [64, 65, 128], [1, 1, 1]), (8, 33, 16, [100, 0, 7], [17, 0, 7]), (2, 64, 128, [300], [300]),
         (1, 65, 64, [70, 80], [70, 2]), (4, 100, 32, [31, 32, 33, 64], [31, 1, 2, 33]), (4, 128, 64, [1000, 3], [999, 3]),
         (16, 40, 16, [16], [16]), (5, 8, 16, [9] * 40, [1] * 40)]


@pytest.mark.parametrize("kv,d,page,lengths,new", CASES)
def test_write_and_read(kv, d, page, lengths, new, dev, ic):
    print(f"[cache] {kv} x {d}, pages of {page}, {lengths} {new}", flush=True)
    rng = np.random.default_rng(kv * 131 + d)
    pages = sum(-(-n // page) for n in lengths) + 3
    held, table = Held(dev, ic, pages, page, kv, d), pages_of(rng, lengths, page, pages, 1)
    start, rows = np.concatenate([[0], np.cumsum(new)]), sum(new) + 2
    k, v = (rng.standard_normal((rows, kv, d)).astype(np.float32) * np.exp(rng.normal(0, 2, (rows, kv, 1))).astype(np.float32)
            for _ in "kv")
    w = kv * d
    s = held.seqs(start, lengths, table)
    # Rows of a packed projection, and of a buffer of their own.
    wide = np.full((rows, 2 * w + 3), np.nan, np.float32)
    wide[:, :w], wide[:, w + 1:2 * w + 1] = k.reshape(rows, w), v.reshape(rows, w)
    X = dev.upload(wide)
    dev.api.ops_cache_write(dev.po, held.p, ic.C.byref(s), rows, ic.mat(X, 0, 2 * w + 3), ic.mat(X, w + 1, 2 * w + 3))
    held.ref.write(k, v, start, lengths, table)
    held.matches()
    # Every kept token back, in one call, and keys or values alone.
    all_start, all_rows = np.concatenate([[0], np.cumsum(lengths)]), sum(lengths) + 1
    t = held.seqs(all_start, lengths, table)
    want = [np.full((all_rows, kv, d), 5, np.float32) for _ in "kv"]
    held.ref.read(all_start, lengths, table, *want)
    for pair in ((1, 1), (1, 0), (0, 1)):
        out = [dev.upload(np.full((all_rows, w + 1), 5, np.float32)) for _ in "kv"]
        dev.api.ops_cache_read(dev.po, held.p, ic.C.byref(t), all_rows,
                               *(ic.Opnd(o.mem if on else None, 0, w + 1, 0, 0) for o, on in zip(out, pair)))
        for o, x, on in zip(out, want, pair):
            got = dev.read(o).reshape(all_rows, w + 1)
            assert np.all(got[:, w] == 5)
            assert np.array_equal(got[:, :w].reshape(x.shape), x if on else np.full_like(x, 5))


def test_no_place(dev, ic):
    """Positions before the first and behind the table, pages given back and
    numbers that are no page, starts past the rows: nothing is written, zeros
    are read."""
    kv, d, page, rows = 2, 24, 16, 40
    rng = np.random.default_rng(1)
    held = Held(dev, ic, 6, page, kv, d)
    table = np.array([[3, -1, 0], [5, 6, -2147483648], [1, 2147483647, 4], [2, 2, 2]], np.int32)
    # Sequence 0: 20 rows over a given back page; 1: more rows than tokens; 2:
    # longer than its table; 3: a length below zero.
    start, length = [0, 20, 26, 36, 39], [44, 4, 50, -5]
    k, v = (rng.standard_normal((rows, kv, d)).astype(np.float32) for _ in "kv")
    s, K, V = held.seqs(start, length, table), dev.upload(k), dev.upload(v)
    w = kv * d
    dev.api.ops_cache_write(dev.po, held.p, ic.C.byref(s), rows, ic.mat(K, 0, w), ic.mat(V, 0, w))
    held.ref.write(k, v, start, length, table)
    held.matches()
    want = [np.full((rows, kv, d), 5, np.float32) for _ in "kv"]
    held.ref.read(start, length, table, *want)
    out = [dev.upload(np.full((rows, kv, d), 5, np.float32)) for _ in "kv"]
    dev.api.ops_cache_read(dev.po, held.p, ic.C.byref(s), rows, *(ic.mat(o, 0, w) for o in out))
    for o, x in zip(out, want):
        assert np.array_equal(dev.read(o).reshape(x.shape), x)
    # Starts out of the rows' range, and lengths at the ends of theirs.
    start, length = [-7, 3, 1000000], [2147483647, 2147483647]
    s = held.seqs(start, length, table[:2])
    dev.api.ops_cache_write(dev.po, held.p, ic.C.byref(s), rows, ic.mat(K, 0, w), ic.mat(V, 0, w))
    held.matches()


def test_values(dev, ic):
    """Rows that are not finite have a scale of NaN and are read as NaN, rows
    of next to nothing as zeros; neighbours keep theirs."""
    kv, d, page = 2, 20, 16
    rng = np.random.default_rng(2)
    k, v = (rng.standard_normal((9, kv, d)).astype(np.float32) for _ in "kv")
    k[1, 0, 3], k[2, 1, 19], v[3, 0, 0] = np.inf, np.nan, -np.inf
    k[4], v[5], k[6], v[7] = 0, 1e-31, 3e38, -1e-40
    held = Held(dev, ic, 2, page, kv, d)
    table = np.array([[1]], np.int32)
    s, K, V = held.seqs([0, 9], [9], table), dev.upload(k), dev.upload(v)
    w = kv * d
    dev.api.ops_cache_write(dev.po, held.p, ic.C.byref(s), 9, ic.mat(K, 0, w), ic.mat(V, 0, w))
    held.ref.write(k, v, [0, 9], [9], table)
    held.matches()
    out, want = [dev.zeros(9 * w) for _ in "kv"], [np.zeros((9, kv, d), np.float32) for _ in "kv"]
    dev.api.ops_cache_read(dev.po, held.p, ic.C.byref(s), 9, *(ic.mat(o, 0, w) for o in out))
    held.ref.read([0, 9], [9], table, *want)
    for o, x in zip(out, want):
        assert np.array_equal(dev.read(o).reshape(x.shape), x, equal_nan=True)


def test_many_sequences_and_far_pages(dev, ic):
    """700 sequences, pages at byte places past 2^31 of the codes."""
    kv, d, page, pages = 8, 128, 128, 17000
    if pages * kv * page * d < 1 << 31:
        pytest.fail("pages end before 2^31")
    rng = np.random.default_rng(3)
    bufs = [dev.alloc(pages * kv * page * n) for n in (d, d, 4, 4)]
    cache = ic.Cache(*(b.mem for b in bufs), pages, page, kv, d)
    n, w = 700, kv * d
    table = (pages - 1 - rng.permutation(n)).astype(np.int32)[:, None]
    length = rng.integers(1, page + 1, n).astype(np.int32)
    k, v = (rng.standard_normal((n, kv, d)).astype(np.float32) for _ in "kv")
    B = [dev.upload(x) for x in (np.arange(n + 1, dtype=np.int32), length, table)]
    s = ic.Seqs(*(b.mem for b in B), n, 1)
    K, V, out = dev.upload(k), dev.upload(v), [dev.zeros(n * w) for _ in "kv"]
    dev.api.ops_cache_write(dev.po, ic.C.byref(cache), ic.C.byref(s), n, ic.mat(K, 0, w), ic.mat(V, 0, w))
    dev.api.ops_cache_read(dev.po, ic.C.byref(cache), ic.C.byref(s), n, *(ic.mat(o, 0, w) for o in out))
    import long_ref as ref
    for o, x in zip(out, (k, v)):
        c, sc = ref.quant(x)
        assert np.array_equal(dev.read(o).reshape(x.shape), c.astype(np.float32) * sc[..., None])
