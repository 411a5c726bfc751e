# SPDX-License-Identifier: Unlicense
"""GPU: rotary positions computed from coordinates against 64 bits.

Both sides form the same 64-bit angle; its remainder rounded to float32 and
the sums of sine and cosine are off by at most 3 U (U = 2^-24) each, the
multiplier, the two products and their difference round once more each: |got
- want| <= 6 U m (|x0| + |x1|)."""

import numpy as np
import pytest

import long_ref as ref
from long_ref import U

pytestmark = pytest.mark.gpu

INTER, INVERSE = 1, 2


def freqs(ic, rot, axes, base=10000.0, kind=0, factor=1.0, trained=4096.0, slow=1.0, fast=32.0):
    f = np.zeros(max(rot // 2, 1))
    if rot:
        ic.api().ops_rope_freqs(f.ctypes.data, rot, axes, base, kind, factor, trained, slow, fast)
    return f[:rot // 2]


# rows, heads, kv heads, d, rot, axes, flags, mult, float offset, pad of a row
SHAPES = [
    (1, 1, 0, 2, 2, 1, 0, 1.0, 0, 0), (1, 16, 4, 128, 128, 1, 0, 1.2, 0, 0), (1, 3, 1, 7, 4, 1, 1, 1.0, 1, 3),
    (5, 2, 2, 64, 64, 2, 1, 1.0, 0, 0), (7, 4, 1, 96, 32, 1, 0, 0.5, 0, 4), (33, 3, 3, 36, 20, 1, 1, 1.0, 2, 2),
    (100, 8, 8, 32, 32, 2, 3, 1.0, 0, 0), (3, 2, 1, 100, 60, 3, 0, 1.0, 4, 8), (41, 1, 1, 128, 64, 1, 2, 1.1, 0, 0),
    (64, 5, 0, 33, 32, 4, 1, 1.0, 3, 1), (2000, 2, 1, 64, 16, 1, 0, 1.0, 0, 0), (9, 2, 2, 40, 0, 1, 0, 1.0, 0, 0),
    (2, 1, 1, 2050, 2048, 1, 0, 1.0, 0, 0), (6, 700, 1, 8, 8, 1, 1, 1.0, 0, 0)]


@pytest.mark.parametrize("place", ["apart", "packed", "in place"])
@pytest.mark.parametrize("shape", SHAPES, ids=[str(s) for s in SHAPES])
def test_edges(shape, place, dev, ic):
    rows, h, kv, d, rot, axes, flags, mult, off, pad = shape
    print(f"[rope pos] {shape} {place}", flush=True)
    rng = np.random.default_rng(rows + d + rot)
    n1, n2 = h * d, kv * d
    ld = n1 + 2 * n2 + pad
    x = rng.standard_normal((rows, ld)).astype(np.float32)
    pos = rng.integers(-50, 100000, (rows, axes)).astype(np.int32)
    f = freqs(ic, rot, axes) if rot % (2 * axes) == 0 else rng.random(rot // 2)
    P, Fq = dev.upload(pos), dev.upload(np.concatenate([f, [0.0]]))
    host = np.concatenate([np.full(off, 5.0), x.ravel(), np.full(4, 5.0)]).astype(np.float32)
    X = dev.upload(host)
    if place == "in place":
        Y1, Y2, l1, l2, o1, o2 = X, X, ld, ld, off, off + n1
    elif place == "packed":
        # Queries and keys side by side, keys first, with a gap.
        l1 = l2 = n1 + n2 + pad
        Y1 = Y2 = dev.upload(np.full(off + rows * l1 + 4, 7.0, np.float32))
        o1, o2 = off + n2, off
    else:
        l1, l2, o1, o2 = n1, max(n2, 1), 0, 0
        Y1, Y2 = (dev.upload(np.full(rows * n + 4, 7.0, np.float32)) for n in (l1, l2))
    dev.api.ops_rope_pos(dev.po, rows, d, rot, axes, P.mem, Fq.mem, mult, flags, ic.mat(X, off, ld),
                         ic.mat(Y1, o1, l1), h, ic.mat(X, off + n1, ld), ic.mat(Y2, o2, l2), kv)
    for name, Y, o, l, a, n in (("q", Y1, o1, l1, 0, h), ("k", Y2, o2, l2, n1, kv)):
        if n == 0:
            continue
        out = dev.read(Y)
        got = out[o:o + (rows - 1) * l + n * d]
        got = np.stack([got[r * l:r * l + n * d] for r in range(rows)]).reshape(rows, n, d)
        xin = x[:, a:a + n * d].reshape(rows, n, d)
        m = float(np.float32(mult))
        want = ref.rope(xin, pos, f, rot, bool(flags & INTER), m, bool(flags & INVERSE))
        assert np.array_equal(got[..., rot:], xin[..., rot:])
        if rot:
            p = np.arange(rot // 2)
            i, j = (2 * p, 2 * p + 1) if flags & INTER else (p, p + rot // 2)
            size = np.abs(xin[..., i]).astype(np.float64) + np.abs(xin[..., j])
            worst = max(np.max(np.abs(got[..., s] - want[..., s]) / (6 * U * m * size + 1e-38)) for s in (i, j))
            print(f"[rope pos] {name} worst {worst:.3f} of the bound", flush=True)
            assert worst <= 1
    if place == "in place":
        out = dev.read(X)
        assert (out[:off] == 5).all() and (out[-4:] == 5).all()
        left = out[off:-4].reshape(rows, ld)
        assert np.array_equal(left[:, n1 + n2:], x[:, n1 + n2:])
    elif place == "packed":
        out = dev.read(Y1)
        rest = out[off:off + rows * l1].reshape(rows, l1)
        assert (out[:off] == 7).all() and (rest[:, n1 + n2:] == 7).all()


def test_grid_as_the_matcher_has_it(dev, ic):
    """Two coordinates, interleaved, 256 channels: the table that the ELoFTR
    driver makes (pair p by row for even p, by column for odd, 10000^(-2 (p /
    2) / 128)), through ops_rope. Its angles are float32: off by U of up to
    20 radians, twice (the frequency, the product)."""
    print("[rope pos] grid", flush=True)
    h = w = 20
    d, n = 256, h * w
    rng = np.random.default_rng(3)
    x = rng.standard_normal((n, d)).astype(np.float32)
    pos = np.stack(np.meshgrid(np.arange(1, h + 1), np.arange(1, w + 1), indexing="ij"), -1).reshape(n, 2)
    p = np.arange(d // 2)
    f32 = (1.0 / 10000.0 ** (2 * (p // 2) / 128)).astype(np.float32)
    a = (pos[:, p % 2].astype(np.float32) * f32).astype(np.float32)
    cs = np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32)
    f = freqs(ic, d, 2)
    assert np.allclose(f, 10000.0 ** (-2 * (p // 2) / 128), rtol=1e-14)
    A, T, P, Fq = dev.upload(x), dev.upload(cs), dev.upload(pos.astype(np.int32)), dev.upload(f)
    Y = dev.zeros(n * d)
    dev.api.ops_rope_pos(dev.po, n, d, d, 2, P.mem, Fq.mem, 1.0, INTER, ic.mat(A, 0, d), ic.mat(Y, 0, d), 1,
                         ic.mat(None, 0, 0), ic.mat(None, 0, 0), 0)
    dev.api.ops_rope(dev.po, A.mem, 0, d, n, 1, d, n, T.mem, 1)
    got, table = (dev.read(b, n * d) for b in (Y, A))
    size = np.abs(x).reshape(n, -1, 2).sum(-1).repeat(2, -1).ravel()
    assert np.all(np.abs(got - table) <= U * (2 * 20 + 12) * size)


@pytest.mark.parametrize("flags", [0, INTER])
def test_far_positions(flags, dev, ic):
    """Positions up to the largest int32, at the trained frequencies."""
    print(f"[rope pos] far {flags}", flush=True)
    d, rows = 64, 40
    rng = np.random.default_rng(9)
    pos = np.concatenate([2 ** 31 - 1 - np.arange(20), -2 ** 31 + np.arange(20)])[:, None]
    x, f = rng.standard_normal((rows, d)).astype(np.float32), freqs(ic, d, 1)
    X, P, Fq, Y = dev.upload(x), dev.upload(pos.astype(np.int32)), dev.upload(f), dev.zeros(rows * d)
    dev.api.ops_rope_pos(dev.po, rows, d, d, 1, P.mem, Fq.mem, 1.0, flags, ic.mat(X, 0, d), ic.mat(Y, 0, d), 1,
                         ic.mat(None, 0, 0), ic.mat(None, 0, 0), 0)
    want = ref.rope(x[:, None], pos, f, d, bool(flags))[:, 0]
    p = np.arange(d // 2)
    i, j = (2 * p, 2 * p + 1) if flags else (p, p + d // 2)
    size = np.zeros((rows, d))
    size[:, i] = size[:, j] = np.abs(x[:, i]).astype(np.float64) + np.abs(x[:, j])
    assert np.all(np.abs(dev.read(Y, rows * d).reshape(rows, d) - want) <= 6 * U * size)


@pytest.mark.parametrize("flags", [0, INTER])
@pytest.mark.parametrize("rot", [48, 20])
def test_gradient(flags, rot, dev, ic):
    """The inverse call on g is the gradient of sum g y by the formula, and by
    differences in 64 bits of what the forward call computes (linear: a
    difference over a step of 1 in each input is the derivative)."""
    print(f"[rope pos] gradient {flags} {rot}", flush=True)
    rows, h, d, m = 3, 2, 48, 1.25
    rng = np.random.default_rng(rot)
    pos = rng.integers(0, 5000, (rows, 1)).astype(np.int32)
    f = freqs(ic, rot, 1)
    g = rng.standard_normal((rows, h, d)).astype(np.float32)
    P, Fq, n = dev.upload(pos), dev.upload(f), rows * h * d

    def call(x, fl):
        X, Y = dev.upload(x.astype(np.float32)), dev.zeros(n)
        dev.api.ops_rope_pos(dev.po, rows, d, rot, 1, P.mem, Fq.mem, m, flags | fl, ic.mat(X, 0, h * d),
                             ic.mat(Y, 0, h * d), h, ic.mat(None, 0, 0), ic.mat(None, 0, 0), 0)
        return dev.read(Y, n).reshape(rows, h, d)

    got = call(g, INVERSE)
    want = ref.rope(g, pos, f, rot, bool(flags), m, True)
    assert np.all(np.abs(got - want) <= 6 * U * m * 2 * np.abs(g).max())
    for c in range(d):
        e = np.zeros((rows, h, d))
        e[..., c] = 1
        # y(e) is column c of the rotation, each entry off by 6 U m at most.
        diff = (g.astype(np.float64) * call(e, 0)).sum(-1)
        assert np.all(np.abs(diff - got[..., c]) <= 6 * U * m * (np.abs(g).sum(-1) + 2 * np.abs(g).max()))


def test_recorded_and_replayed(dev, ic):
    """A decoding step's rotation in place in a packed row: recorded once,
    replayed as the position and the row change."""
    print("[rope pos] graph", flush=True)
    h, kv, d = 8, 2, 64
    ld = (h + 2 * kv) * d
    f = freqs(ic, d, 1, kind=3, factor=8.0)
    X, P, Fq = dev.zeros(ld), dev.upload(np.zeros(1, np.int32)), dev.upload(f)
    dev.api.ocl_graph_begin(dev.pb)
    dev.api.ops_rope_pos(dev.po, 1, d, d, 1, P.mem, Fq.mem, 1.2, 0, ic.mat(X, 0, ld), ic.mat(X, 0, ld), h,
                         ic.mat(X, h * d, ld), ic.mat(X, h * d, ld), kv)
    graph = dev.api.ocl_graph_end(dev.pb)
    try:
        for t in range(4):
            x = np.random.default_rng(t).standard_normal(ld).astype(np.float32)
            dev.write(X, x)
            dev.write(P, np.array([1000 * t + 1], np.int32))
            dev.api.ocl_graph_launch(dev.pb, graph)
            got = dev.read(X, ld).reshape(-1, d)
            m = float(np.float32(1.2))
            want = ref.rope(x[:(h + kv) * d].reshape(1, -1, d), np.array([[1000 * t + 1]]), f, d, False, m)[0]
            size = np.abs(x.reshape(-1, 2, d // 2)).astype(np.float64).sum(1)
            size = np.concatenate([size, size], 1)[:h + kv]
            assert np.all(np.abs(got[:h + kv] - want) <= 6 * U * m * size)
            assert np.array_equal(got[h + kv:].ravel(), x[(h + kv) * d:])
    finally:
        ic.lib().ocl_graph_free(graph)
