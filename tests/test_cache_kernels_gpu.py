# SPDX-License-Identifier: Unlicense
"""GPU: the cache's kernels that move four heads at a time, which calls of many
rows take, to the bit like the others: every width of a group of lanes, heads
that are left over, rows without a place and of no sequence."""

import numpy as np
import pytest

from test_cache_gpu import Held, pages_of

pytestmark = pytest.mark.gpu

# Key heads, channels, page.
SHAPES = [(4, 8, 16), (5, 24, 32), (8, 32, 16), (11, 30, 64), (6, 40, 16), (8, 64, 64), (9, 33, 32), (4, 63, 128), (7, 100, 32),
          (4, 128, 64), (5, 65, 16), (8, 127, 128)]


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("kv,d,page", SHAPES)
def test_many_rows(kv, d, page, four, dev, ic):
    lanes = 8 if d <= 32 else 16 if d <= 64 else 32
    # The first number of rows that fills the CUs twice, and the one before it.
    rows = -(-512 * dev.ocl.cu_count // (kv * lanes)) - (not four)
    print(f"[cache] {rows} rows of {kv} x {d}, pages of {page}", flush=True)
    assert kv >= 4 and (rows * kv * lanes >= 512 * dev.ocl.cu_count) == four
    rng = np.random.default_rng(kv * 131 + d + four)
    new = [rows // 3, 0, 1, rows // 2 - 20]
    lengths = [new[0] + 40, 30, 9, new[3] - 5]
    pages = sum(-(-n // page) for n in lengths) + 3
    held, table = Held(dev, ic, pages, page, kv, d), pages_of(rng, lengths, page, pages, 4)
    # Pages given back, and numbers of none.
    table[0, 2], table[0, 5], table[3, 1], table[3, 4] = -1, pages, 2147483647, -5
    # Rows before the first sequence, and behind the last.
    start = np.concatenate([[0], np.cumsum(new)]) + 7
    assert start[-1] < rows
    k, v = (rng.standard_normal((rows, kv, d)).astype(np.float32) * np.exp(rng.normal(0, 2, (rows, kv, 1))).astype(np.float32)
            for _ in "kv")
    k[9, kv - 1, d - 1], v[11, 0, 0], k[13], v[14, kv // 2] = np.nan, np.inf, 0, 1e-35
    w, ld = kv * d, 2 * kv * d + 3
    wide = np.full((rows, ld), np.nan, np.float32)
    wide[:, :w], wide[:, w + 1:2 * w + 1] = k.reshape(rows, w), v.reshape(rows, w)
    X, s = dev.upload(wide), held.seqs(start, lengths, table)
    dev.api.ops_cache_write(dev.po, held.p, ic.C.byref(s), rows, ic.mat(X, 0, ld), ic.mat(X, w + 1, ld))
    held.ref.write(k, v, start, lengths, table)
    held.matches()
    want = [np.full((rows, kv, d), 5, np.float32) for _ in "kv"]
    held.ref.read(start, lengths, table, *want)
    for pair in ((1, 1), (1, 0), (0, 1)):
        out = [dev.upload(np.full((rows, w + 1), 5, np.float32)) for _ in "kv"]
        dev.api.ops_cache_read(dev.po, held.p, ic.C.byref(s), rows,
                               *(ic.Opnd(o.mem if on else None, 0, w + 1, 0, 0) for o, on in zip(out, pair)))
        for o, x, on in zip(out, want, pair):
            got = dev.read(o).reshape(rows, w + 1)
            assert np.all(got[:, w] == 5)
            assert np.array_equal(got[:, :w].reshape(x.shape), x if on else np.full_like(x, 5), equal_nan=True)
