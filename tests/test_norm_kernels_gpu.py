# SPDX-License-Identifier: Unlicense
"""GPU: ops_rms_norm at the sizes where its kernels and launches change hands,
to the bit as the definition has it."""

import numpy as np
import pytest

import kept_ref
from test_norm_gpu import check, data, run

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


def lanes_sum(v):
    """A wave's sum of its 64 lanes' values (..., 64)."""
    for order in (lambda i: i ^ 1, lambda i: i ^ 2, lambda i: i ^ 7, lambda i: i ^ 15):
        v = v + v[..., order(np.arange(64))]
    return (v[..., 0] + v[..., 16]) + (v[..., 32] + v[..., 48])


def inverse(x, eps, ahead):
    """1 / rms as float32, the squares added 256 channels at a time or, with
    `ahead`, a lane's through the row in steps of 256 `ahead` channels first."""
    blocks = -(-x.shape[1] // 256)
    sq = np.zeros((len(x), -(-blocks // 16) * 16, 64, 4))
    sq.reshape(len(x), -1)[:, :x.shape[1]] = x.astype(np.float64) ** 2
    if ahead:
        wave = np.zeros((len(x), ahead, 64))
        for k in range(0, sq.shape[1], ahead):
            for j in range(4):
                wave += sq[:, k:k + ahead, :, j]
    else:
        wave = np.zeros(sq.shape[:3])
        for j in range(4):
            wave += sq[..., j]
    total = np.zeros(len(x))
    for b in lanes_sum(wave).T:
        total = total + b
    return (1 / np.sqrt(total / x.shape[1] + np.float64(np.float32(eps)))).astype(np.float32)


def rows_at_a_border(c, count, eps=1e-6):
    """Rows whose 1 / rms lies so near the middle of two floats that the order
    of the sum decides: three channels are set so that it does."""
    rng, rows = np.random.default_rng(c), []
    while len(rows) < count:
        x = rng.standard_normal((4000, c)).astype(np.float32)
        x[:, :3] = 0
        sum3 = (x.astype(np.float64) ** 2).sum(1)
        near = (1 / np.sqrt((sum3 + 4) / c + np.float64(np.float32(eps)))).astype(np.float32)
        middle = (near.astype(np.float64) + np.nextafter(near, np.float32(0)).astype(np.float64)) / 2
        want = c * (1 / middle ** 2 - np.float64(np.float32(eps))) * (1 + 2.0 ** -53 * rng.integers(-8, 9, len(x)))
        for j in range(3):
            left = want - (x.astype(np.float64) ** 2).sum(1)
            root = np.sqrt(np.maximum(left, 0)).astype(np.float32)
            x[:, j] = np.where(root.astype(np.float64) ** 2 > left, np.nextafter(root, np.float32(0)), root)
        found = np.flatnonzero(inverse(x, eps, 0) != inverse(x, eps, 1 if c <= 1024 else 4))
        rows += list(x[found[:count - len(rows)]])
    return np.array(rows)


@pytest.mark.parametrize("c,many", [(300, 2560), (1024, 3000), (1500, 384), (4096, 500)])
def test_same_from_every_kernel(c, many, dev, ic):
    """A row among many has the bits that it has alone, where the order of the
    sum of squares decides how its mean is rounded."""
    x = rows_at_a_border(c, 8)
    alone = run(dev, ic, x)
    among = run(dev, ic, np.concatenate([x, np.ones((many - len(x), c), np.float32)]))
    for k in ("y", "q", "s"):
        assert np.array_equal(alone[k], among[k][:len(x)]), k


# Both sides of where kernels change hands, by rows and by channels, with parts
# of a step of 4, 256 and 1024 channels left over.
@pytest.mark.parametrize("n,c", [(2559, 1024), (2560, 1024), (2561, 257), (2600, 513), (3202, 1023), (2559, 300), (383, 4096),
                                 (384, 4096), (400, 1025), (500, 4093), (600, 2049), (383, 3000), (300, 4097), (200, 16384)])
def test_many_rows_of_every_width(n, c, dev, ic):
    print(f"[norm] {n} x {c}", flush=True)
    x, r, g = data(n, c)
    check(run(dev, ic, x, r, g), x, r, g)
    check(run(dev, ic, x, r, g, pads=(3, 1, 64, 2)), x, r, g)
    check(run(dev, ic, x, None, None, h=False), x, None, None)
    check(run(dev, ic, x, r, g, y=False), x, r, g)
    check(run(dev, ic, x, r, g, q=False), x, r, g)
    for alias in ([("h", "x")], [("h", "r"), ("y", "x")], [("y", "r")]):
        check(run(dev, ic, x, r, g, alias=alias), x, r, g)


@pytest.mark.parametrize("n,c", [(2560, 700), (390, 4000), (400, 4096)])
def test_values_among_many_rows(n, c, dev, ic):
    """Zeros, magnitudes whose squares pass float32's range, subnormal ones and
    values that are not finite, each in rows of its own."""
    x, _, g = data(n, c)
    x[0] = 0
    x[1] = 1e30 * np.sign(x[1])
    x[2] *= np.float32(1e-30)
    x[3] = np.float32(1e-42)
    x[4, c // 2], x[n - 1, c - 1], x[5, 0] = np.inf, -np.inf, np.nan
    x[6, 1:] = 0
    for eps in (1e-6, 1e-45):
        check(run(dev, ic, x, None, g, eps), x, None, g, eps)
