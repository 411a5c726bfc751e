# SPDX-License-Identifier: Unlicense
"""GPU: ops_rms_norm at the sizes where its kernels and launches change hands,
to the bit as the definition has it."""

import numpy as np
import pytest

import kept_ref

pytestmark = pytest.mark.gpu


def test_wide_rows_of_several_launches(dev, ic):
    """More rows of more than 4096 channels (1024 threads each) than have 2^32
    threads: 69 GB in place, random ones around where launches may end."""
    n, c = (1 << 22) + 3, 4097
    X = dev.alloc(4 * n * c)
    dev.api.ocl_fill(dev.pb, X.mem, 0, n * c, 2.0)
    rng = np.random.default_rng(0)
    some = {at: rng.standard_normal((3, c)).astype(np.float32) for at in (0, (1 << 20) - 1, (1 << 21) - 1, 3 * (1 << 20) - 1,
                                                                          (1 << 22) - 3, n - 3)}
    for at, x in some.items():
        dev.write(X, x, 4 * at * c)
    none, rows = ic.Opnd(None, 0, 0, 0, 0), ic.mat(X, 0, c)
    print("[norm] 69 GB", flush=True)
    dev.api.ops_rms_norm(dev.po, n, c, rows, none, None, 1e-6, none, rows, None, None)
    written = {at + i: x[i] for at, x in some.items() for i in range(3)}
    same = np.full((1, c), 2, np.float32)
    for at in [*written, 5, 1000000, (1 << 21) + 7, (1 << 22) - 9]:
        x = written[at][None] if at in written else same
        got = dev.read(X, c, off_bytes=4 * at * c)
        assert np.array_equal(got, kept_ref.rms_norm(x, None, None, 1e-6)[1][0]), at
