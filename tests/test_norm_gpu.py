# SPDX-License-Identifier: Unlicense
"""GPU: ops_rms_norm against its definition, whose sums, codes and scales are
defined to the bit: no tolerance."""

import numpy as np
import pytest

import kept_ref
import long_ref as ref

pytestmark = pytest.mark.gpu

# Rows, channels: one to many, around 256, 1024, 4096 and 16384, where another
# kernel takes over, odd ones.
SIZES = [(1, 1), (1, 3), (5, 64), (3, 65), (2, 255), (7, 256), (9, 257), (1, 1000), (33, 1023), (2, 1024), (1, 1024),
         (5, 1025), (130, 768), (2, 4095), (3, 4096), (1, 4096), (2, 4097), (1, 16384), (2, 16385), (1, 40001), (700, 100)]


def run(dev, ic, x, r=None, g=None, eps=1e-6, h=True, y=True, q=True, pads=(0, 0, 0, 0), alias=None):
    """The call's outputs as arrays; `pads`: floats between the rows of x, r,
    h, y; `alias` (output, input): the output lies over the input."""
    n, c = x.shape
    ld = dict(zip("xrhy", (c + p for p in pads)))
    bufs = {}
    for name, a in (("x", x), ("r", r)):
        if a is not None:
            wide = np.full((n, ld[name]), np.nan, np.float32)
            wide[:, :c] = a
            bufs[name] = dev.upload(wide)
    for name, want in (("h", h), ("y", y)):
        if want:
            bufs[name] = dev.upload(np.full((n, ld[name]), 7, np.float32))
    for out, inp in alias or ():
        bufs[out], ld[out] = bufs[inp], ld[inp]
    op = lambda k: ic.Opnd(bufs[k].mem if k in bufs else None, 0, ld[k], 0, 0)  # noqa: E731
    G = dev.upload(g) if g is not None else None
    Q = dev.upload(np.full(n * ref.pitch(c), 99, np.int8)) if q else None
    S = dev.upload(np.full(n, 99, np.float32)) if q else None
    dev.api.ops_rms_norm(dev.po, n, c, op("x"), op("r"), ic.mem(G), eps, op("h"), op("y"), ic.mem(Q), ic.mem(S))
    got = {}
    for name in "hy":
        if name in bufs and (h if name == "h" else y):
            wide = dev.read(bufs[name], n * ld[name]).reshape(n, ld[name])
            got[name] = wide[:, :c]
            if not alias:
                assert np.all(wide[:, c:] == 7)
    if q:
        got["q"] = dev.read(Q, n * ref.pitch(c), np.int8).reshape(n, -1)
        got["s"] = dev.read(S, n)
    return got


def check(got, x, r, g, eps=1e-6):
    h, y = kept_ref.rms_norm(x, r, g, eps)
    if "h" in got:
        assert np.array_equal(got["h"], h, equal_nan=True)
    if "y" in got:
        assert np.array_equal(got["y"], y, equal_nan=True)
    if "q" in got:
        c, s = ref.quant(y)
        assert np.array_equal(got["s"], s, equal_nan=True)
        assert np.array_equal(got["q"][:, :x.shape[1]], c) and not got["q"][:, x.shape[1]:].any()


def data(n, c, seed=0):
    rng = np.random.default_rng(n * 7919 + c + seed)
    x, r = (rng.standard_normal((n, c)).astype(np.float32) * np.exp(rng.normal(0, 2, (n, 1))).astype(np.float32)
            for _ in "xr")
    return x, r, (1 + 0.3 * rng.standard_normal(c)).astype(np.float32)


@pytest.mark.parametrize("n,c", SIZES)
def test_all_outputs(n, c, dev, ic):
    print(f"[norm] {n} x {c}", flush=True)
    x, r, g = data(n, c)
    check(run(dev, ic, x, r, g), x, r, g)


@pytest.mark.parametrize("n,c", [(3, 70), (5, 1024), (2, 4100), (1, 17000)])
def test_each_output_alone(n, c, dev, ic):
    x, r, g = data(n, c)
    for h, y, q in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (0, 1, 1), (1, 1, 0)):
        check(run(dev, ic, x, r, g, h=h, y=y, q=q), x, r, g)
    check(run(dev, ic, x, None, g), x, None, g)
    check(run(dev, ic, x, r, None), x, r, None)
    check(run(dev, ic, x, None, None, h=False), x, None, None)


@pytest.mark.parametrize("n,c", [(5, 100), (4, 1024), (3, 4096), (3, 16390)])
def test_strides_and_places(n, c, dev, ic):
    x, r, g = data(n, c)
    check(run(dev, ic, x, r, g, pads=(1, 4, 3, 64)), x, r, g)
    for alias in ([("h", "x")], [("h", "r")], [("y", "x")], [("h", "r"), ("y", "x")], [("h", "x"), ("y", "r")]):
        check(run(dev, ic, x, r, g, alias=alias), x, r, g)


@pytest.mark.parametrize("c", [60, 1024, 4096, 20000])
def test_values(c, dev, ic):
    """Zeros, magnitudes whose squares pass float32's range, subnormal ones, a
    value that is not finite: its row alone is NaN."""
    x, _, g = data(9, c)
    x[0] = 0
    x[1] = 1e30 * np.sign(x[1])
    x[2] *= np.float32(1e-30)
    x[3] = np.float32(1e-42)
    x[4, c // 2] = np.inf
    x[5, 0] = np.nan
    x[6, 1:] = 0
    x[7] = 2.0 ** 60
    for eps in (1e-6, 1e-38, 1e-45):
        check(run(dev, ic, x, None, g, eps), x, None, g, eps)
    check(run(dev, ic, x, -x, g, 1e-45), x, -x, g, 1e-45)


def test_many_rows(dev, ic):
    x, r, g = data(70001, 16)
    check(run(dev, ic, x, r, g), x, r, g)


def test_graph(dev, ic):
    """Recorded and replayed on new values, beside eager calls."""
    n, c = 33, 1024
    x, r, g = data(n, c)
    X, R, G, Y = dev.upload(x), dev.upload(r), dev.upload(g), dev.zeros(n * c)
    Q, S = dev.alloc(n * c), dev.zeros(n)
    none = ic.Opnd(None, 0, 0, 0, 0)

    def call():
        dev.api.ops_rms_norm(dev.po, n, c, ic.mat(X, 0, c), ic.mat(R, 0, c), G.mem, 1e-6, none, ic.mat(Y, 0, c), Q.mem,
                             S.mem)
    dev.api.ocl_graph_begin(dev.pb)
    call()
    graph = dev.api.ocl_graph_end(dev.pb)
    try:
        for seed in range(3):
            x, r, _ = data(n, c, seed + 1)
            dev.write(X, x)
            dev.write(R, r)
            dev.api.ocl_graph_launch(dev.pb, graph)
            check({"y": dev.read(Y).reshape(n, c), "q": dev.read(Q, n * c, np.int8).reshape(n, c), "s": dev.read(S, n)},
                  x, r, g)
            call()
            dev.finish()
    finally:
        ic.lib().ocl_graph_free(graph)


def test_rows_of_two_launches(dev, ic):
    """More rows than one launch takes."""
    n = (1 << 22) + 5
    x, g = np.random.default_rng(4).standard_normal((n, 4), dtype=np.float32), np.array([1, 0.5, 2, -3], np.float32)
    check(run(dev, ic, x, None, g, h=False), x, None, g)
