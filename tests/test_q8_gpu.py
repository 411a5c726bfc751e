# SPDX-License-Identifier: Unlicense
"""GPU: 8-bit rows and linear layers on them against their definition.

The codes and scales are equal to the bit: float32 quotients and products are
rounded as IEEE has it on both sides. The product's whole-number sum is
exact; its conversion, the product of the scales, theirs, the bias and the
residual round once each, at most U = 2^-24 of what they give: |got - want|
<= U (3 |v| + |v + b| + |y|) for v = sx sw sum, plus what an activation adds: a
gradient of at most 1.13 on the error before it, and 8 U of |v + b| for erff,
tanhf and the products around them."""

import numpy as np
import pytest

import long_ref as ref
from long_ref import U

pytestmark = pytest.mark.gpu


def codes(dev, ic, x, off=0, ld=None):
    """ops_quant_rows of x's rows at float offset off, row stride ld."""
    rows, C = x.shape
    ld = C if ld is None else ld
    host = np.full(off + rows * ld + 4, 9.0, np.float32)
    for r in range(rows):
        host[off + r * ld:off + r * ld + C] = x[r]
    X, p = dev.upload(host), ref.pitch(C)
    assert dev.api.ops_q8_pitch(C) == p
    Q = dev.upload(np.full(rows * p + 64, 77, np.int8))
    S = dev.upload(np.full(rows + 4, 5.0, np.float32))
    dev.api.ops_quant_rows(dev.po, rows, C, X.mem, off, ld, Q.mem, S.mem)
    q, s = dev.read(Q, rows * p + 64, np.int8), dev.read(S)
    assert (q[rows * p:] == 77).all() and (s[rows:] == 5).all()
    return Q, S, q[:rows * p].reshape(rows, p), s[:rows]


@pytest.mark.parametrize("rows,C,off,pad", [
    (1, 1, 0, 0), (5, 3, 1, 2), (3, 63, 0, 0), (130, 64, 0, 64), (7, 65, 0, 3), (9, 255, 2, 0),
    (4, 256, 0, 0), (6, 257, 0, 0), (33, 1000, 4, 4), (5, 1024, 0, 0), (2, 4096, 0, 0),
    (3, 4100, 0, 0), (1, 5001, 0, 0), (2, 131072, 0, 0)])
def test_codes(rows, C, off, pad, dev, ic):
    print(f"[q8] codes {rows} {C} {off} {pad}", flush=True)
    rng = np.random.default_rng(C)
    x = (rng.standard_normal((rows, C)) * np.exp2(rng.integers(-60, 60, (rows, 1)))).astype(np.float32)
    if C >= 8:
        # Ties of every parity: 127 / a = 1, products k + 1/2.
        x[0, :8] = [127, 0.5, 1.5, 2.5, -0.5, -1.5, -126.5, 126.5]
        x[0, 8:] = 0
    _, _, q, s = codes(dev, ic, x, off, C + pad)
    c, want = ref.quant(x)
    assert np.array_equal(s, want)
    assert np.array_equal(q[:, :C], c) and not q[:, C:].any()


def test_codes_of_special_rows(dev, ic):
    """Zeros, rows below and at the smallest maximum, the largest values,
    subnormal ones, infinities and NaN of either sign."""
    print("[q8] special rows", flush=True)
    x = np.zeros((9, 100), np.float32)
    x[1] = 1e-40
    x[2, 5] = np.nextafter(np.float32(2.0 ** -100), np.float32(0))
    x[3, 5], x[3, 6] = 2.0 ** -100, -2.0 ** -101
    x[4, ::2], x[4, 1] = 3.4028235e38, -1.7e38
    x[5, 3], x[5, 4] = np.inf, 1
    x[6, 99] = np.nan
    x[7, 0] = -np.nan
    x[8, 50] = -np.inf
    _, _, q, s = codes(dev, ic, x)
    c, want = ref.quant(x)
    assert np.array_equal(s, want, equal_nan=True) and np.isnan(want[5:]).all()
    assert np.array_equal(q[:, :100], c)
    assert not c[:3].any() and c[3, 5] == 127 and c[4, 0] == 127


# rows, in, out, act, bias, residual (1: other buffer, 2: in place), offsets
# and strides beyond the packed ones
SHAPES = [
    (1, 1, 1, 0, 0, 0, 0), (1, 1024, 4096, 1, 1, 0, 0), (1, 100, 37, 0, 1, 1, 1), (2, 64, 1, 2, 0, 2, 0),
    (3, 513, 129, 4, 1, 0, 3), (4, 4096, 300, 0, 0, 0, 0), (5, 64, 64, 0, 0, 0, 0), (8, 200, 1000, 3, 1, 1, 1),
    (16, 320, 77, 0, 1, 2, 2), (17, 1000, 256, 1, 1, 0, 0), (64, 192, 64, 0, 1, 0, 0), (65, 128, 65, 0, 0, 1, 1),
    (127, 300, 129, 2, 1, 0, 0), (400, 256, 256, 0, 0, 0, 0), (333, 517, 1001, 4, 1, 1, 5),
    (1601, 1024, 1024, 0, 1, 2, 0), (785, 2048, 900, 1, 1, 0, 0), (3202, 1024, 2049, 0, 1, 0, 0),
    (6000, 320, 6100, 0, 1, 0, 0), (4000, 100, 4097, 0, 1, 1, 3), (6400, 192, 1024, 1, 1, 0, 0),
    (3100, 260, 1028, 0, 0, 1, 4), (40, 700, 530, 1, 1, 2, 2), (9000, 64, 1000, 0, 1, 0, 0),
    (60, 300, 4100, 1, 1, 0, 4), (200, 4096, 1500, 0, 0, 0, 0)]


def operands(shape, seed=0):
    rows, cin, cout, act, bias, res, pad = shape
    rng = np.random.default_rng(rows + cin + cout + seed)
    x = rng.standard_normal((rows, cin)).astype(np.float32)
    w = (rng.standard_normal((cout, cin)) / cin ** 0.5).astype(np.float32)
    b = rng.standard_normal(cout).astype(np.float32) if bias else None
    r = rng.standard_normal((rows, cout)).astype(np.float32) if res else None
    return x, w, b, r


def expected(x, w, b, r, kind, slope):
    (xc, xs), (wc, ws) = ref.quant(x), ref.quant(w)
    v = (xc.astype(np.float64) @ wc.astype(np.float64).T) * xs[:, None].astype(np.float64) * ws.astype(np.float64)
    t = v + (0 if b is None else b.astype(np.float64))
    y = ref.act(t, kind, slope)
    want = y + (0 if r is None else r.astype(np.float64))
    grow, own = (1.13, 8) if kind in (1, 4) else (1, 1)
    bound = U * (grow * (3 * np.abs(v) + np.abs(t)) + own * np.abs(t) + np.abs(y) + np.abs(want)) + 1e-37
    return want, bound


def strided(dev, y, off, ld, fill=7.0):
    rows, n = y.shape
    host = np.full(off + rows * ld + 8, fill, np.float32)
    view = host[off:off + rows * ld].reshape(rows, ld)
    view[:, :n] = y
    return dev.upload(host)


def test_every_kernel_is_among_the_shapes(dev, ic):
    """The shapes below reach every kernel, and one is cut by tokens."""
    got, cut = set(), 0
    for rows, cin, cout, *_ in SHAPES:
        while rows:
            n = ic.C.c_int()
            got.add(ic.lib().icoreg_q8_choice(dev.po, rows, cin, cout, ic.C.byref(n)))
            cut += n.value < rows
            rows -= n.value
    assert got == set(range(6)) and cut


@pytest.mark.parametrize("entry", ["q8", "qq"])
@pytest.mark.parametrize("shape", SHAPES, ids=[str(s) for s in SHAPES])
def test_linear(shape, entry, dev, ic):
    rows, cin, cout, act, bias, res, pad = shape
    print(f"[q8] {entry} {shape}", flush=True)
    x, w, b, r = operands(shape)
    want, bound = expected(x, w, b, r, act, 0.25)
    W = dev.upload(w)
    WQ, WS = dev.alloc(cout * ref.pitch(cin)), dev.alloc(cout * 4)
    dev.api.ops_quant_rows(dev.po, cout, cin, W.mem, 0, cin, WQ.mem, WS.mem)
    B = dev.upload(b) if bias else None
    ldx, ldy = cin + pad, cout + pad
    X, Y = strided(dev, x, pad, ldx), strided(dev, r if res == 2 else np.full((rows, cout), 3.0), pad, ldy)
    R = Y if res == 2 else strided(dev, r, pad, ldy, -1.0) if res else None
    if entry == "q8":
        n = dev.api.ops_linear_q8_work_bytes(rows, cin)
        work = dev.upload(np.full(n + 16, 0x55, np.uint8))
        dev.api.ops_linear_q8(dev.po, rows, cin, cout, X.mem, pad, ldx, WQ.mem, WS.mem, ic.mem(B), ic.mem(R), pad,
                              Y.mem, pad, ldy, act, 0.25, work.mem)
        assert (dev.read(work, 16, np.uint8, n) == 0x55).all()
    else:
        XQ, XS = dev.alloc(rows * ref.pitch(cin)), dev.alloc(rows * 4)
        dev.api.ops_quant_rows(dev.po, rows, cin, X.mem, pad, ldx, XQ.mem, XS.mem)
        dev.api.ops_linear_qq(dev.po, rows, cin, cout, XQ.mem, XS.mem, WQ.mem, WS.mem, ic.mem(B), ic.mem(R), pad,
                              Y.mem, pad, ldy, act, 0.25)
    out = dev.read(Y)
    got = out[pad:pad + rows * ldy].reshape(rows, ldy)
    worst = np.max(np.abs(got[:, :cout] - want) / bound)
    print(f"[q8] worst {worst:.3f} of the bound", flush=True)
    assert worst <= 1
    # What lies before, between and behind the rows is as it was.
    assert (out[:pad] == 7).all() and (got[:, cout:] == 7).all() and (out[pad + rows * ldy:] == 7).all()


@pytest.mark.parametrize("rows", [1, 3, 40, 200])
def test_longest_sums(rows, dev, ic):
    """2^17 products of 127^2, of one sign and of both: 2114060288 of 2^31."""
    print(f"[q8] longest sums {rows}", flush=True)
    cin, cout = 131072, 70
    x, w = np.full((rows, cin), 127.0, np.float32), np.full((cout, cin), -127.0, np.float32)
    x[rows // 2, 7:] *= -1
    w[3] *= -1
    w[5, 1000:66000] *= -1
    X, W, Y = dev.upload(x), dev.upload(w), dev.zeros(rows * cout)
    WQ, WS = dev.alloc(cout * cin), dev.alloc(cout * 4)
    work = dev.alloc(dev.api.ops_linear_q8_work_bytes(rows, cin))
    dev.api.ops_quant_rows(dev.po, cout, cin, W.mem, 0, cin, WQ.mem, WS.mem)
    dev.api.ops_linear_q8(dev.po, rows, cin, cout, X.mem, 0, cin, WQ.mem, WS.mem, None, None, 0, Y.mem, 0, cout, 0,
                          0.0, work.mem)
    want = (x.astype(np.float64) @ w.astype(np.float64).T).astype(np.float32)
    assert np.array_equal(dev.read(Y, rows * cout).reshape(rows, cout), want)


@pytest.mark.parametrize("rows", [1, 4, 100])
def test_rows_that_are_not_finite(rows, dev, ic):
    """A token or a weight row with a value that is not finite makes its row or
    column NaN, and nothing else."""
    print(f"[q8] not finite {rows}", flush=True)
    cin, cout = 96, 80
    x, w, _, _ = operands((rows, cin, cout, 0, 0, 0, 0), 1)
    base, _ = expected(x, w, None, None, 0, 0)
    x[0, 3], w[5, 7], w[6, 0] = np.inf, np.nan, -np.inf
    X, W, Y = dev.upload(x), dev.upload(w), dev.zeros(rows * cout)
    WQ, WS = dev.alloc(cout * ref.pitch(cin)), dev.alloc(cout * 4)
    work = dev.alloc(dev.api.ops_linear_q8_work_bytes(rows, cin))
    dev.api.ops_quant_rows(dev.po, cout, cin, W.mem, 0, cin, WQ.mem, WS.mem)
    dev.api.ops_linear_q8(dev.po, rows, cin, cout, X.mem, 0, cin, WQ.mem, WS.mem, None, None, 0, Y.mem, 0, cout, 0,
                          0.0, work.mem)
    got = dev.read(Y, rows * cout).reshape(rows, cout)
    assert np.isnan(got[0]).all() and np.isnan(got[:, 5:7]).all()
    keep = np.delete(np.arange(cout), [5, 6])
    assert np.allclose(got[1:, keep], base[1:, keep], rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("rows", [1, 6, 300])
def test_recorded_and_replayed(rows, dev, ic):
    """A recorded call replayed on other inputs, between eager calls of it."""
    print(f"[q8] graph {rows}", flush=True)
    cin, cout = 512, 640
    x, w, b, _ = operands((rows, cin, cout, 1, 1, 0, 0))
    X, W, B, Y = dev.upload(x), dev.upload(w), dev.upload(b), dev.zeros(rows * cout)
    WQ, WS = dev.alloc(cout * cin), dev.alloc(cout * 4)
    work = dev.alloc(dev.api.ops_linear_q8_work_bytes(rows, cin))

    def call():
        dev.api.ops_linear_q8(dev.po, rows, cin, cout, X.mem, 0, cin, WQ.mem, WS.mem, B.mem, None, 0, Y.mem, 0, cout,
                              1, 0.0, work.mem)

    dev.api.ops_quant_rows(dev.po, cout, cin, W.mem, 0, cin, WQ.mem, WS.mem)
    dev.api.ocl_graph_begin(dev.pb)
    call()
    graph = dev.api.ocl_graph_end(dev.pb)
    try:
        for seed in range(4):
            x = np.random.default_rng(seed).standard_normal((rows, cin)).astype(np.float32)
            dev.write(X, x)
            call()
            eager = dev.read(Y)
            dev.api.ocl_fill(dev.pb, Y.mem, 0, rows * cout, 0.0)
            dev.api.ocl_graph_launch(dev.pb, graph)
            assert np.array_equal(dev.read(Y), eager)
            want, bound = expected(x, w, b, None, 1, 0)
            assert np.all(np.abs(eager.reshape(rows, cout) - want) <= bound)
    finally:
        ic.lib().ocl_graph_free(graph)


# Tokens, channels in and out: blocks of 16 and of 32 tokens that code their
# tokens themselves and that do not, then each tile of the product.
INFINITE = [(1, 96, 80), (20, 1000, 130), (400, 256, 256), (200, 300, 700), (785, 128, 1000), (1800, 64, 2100),
            (2100, 64, 2100), (2000, 96, 4100)]


def test_every_kernel_is_among_the_infinite_sums(dev, ic):
    assert {ic.lib().icoreg_q8_choice(dev.po, *s, None) for s in INFINITE} == set(range(6))


@pytest.mark.parametrize("entry", ["q8", "qq"])
@pytest.mark.parametrize("act", range(5))
@pytest.mark.parametrize("shape", INFINITE, ids=[str(s) for s in INFINITE])
def test_infinite_sums(shape, act, entry, dev, ic):
    """Finite tokens and weights, biases of either infinity and a token and two
    channels whose products pass float32's range: the activations' own
    values there, as the definition has them (ReLU of minus infinity is 0,
    GELU of plus infinity infinity, of minus infinity minus infinity times 0). A
    token that is not finite stays NaN through each of them. Every other output
    is within its bound."""
    print(f"[q8] infinite sums {entry} {shape} {act}", flush=True)
    rows, cin, cout = shape
    x, w, b, _ = operands((rows, cin, cout, act, 1, 0, 0), 2)
    x[0] *= 2.0 ** 100
    w[2] *= 2.0 ** 60
    w[3] = -w[2]
    b[[0, 17]], b[[1, cout - 1]] = np.inf, -np.inf
    if rows > 1:
        x[-1, 5] = np.nan
    X, W, B, Y = dev.upload(x), dev.upload(w), dev.upload(b), dev.zeros(rows * cout)
    WQ, WS = dev.alloc(cout * ref.pitch(cin)), dev.alloc(cout * 4)
    dev.api.ops_quant_rows(dev.po, cout, cin, W.mem, 0, cin, WQ.mem, WS.mem)
    if entry == "q8":
        work = dev.alloc(dev.api.ops_linear_q8_work_bytes(rows, cin))
        dev.api.ops_linear_q8(dev.po, rows, cin, cout, X.mem, 0, cin, WQ.mem, WS.mem, B.mem, None, 0, Y.mem, 0, cout,
                              act, 0.25, work.mem)
    else:
        XQ, XS = dev.alloc(rows * ref.pitch(cin)), dev.alloc(rows * 4)
        dev.api.ops_quant_rows(dev.po, rows, cin, X.mem, 0, cin, XQ.mem, XS.mem)
        dev.api.ops_linear_qq(dev.po, rows, cin, cout, XQ.mem, XS.mem, WQ.mem, WS.mem, B.mem, None, 0, Y.mem, 0, cout,
                              act, 0.25)
    got = dev.read(Y, rows * cout).reshape(rows, cout)
    some = np.unique(np.r_[0:min(rows, 16), rows - 1, np.random.default_rng(rows).integers(0, rows, 24)])
    (xc, xs), (wc, ws) = ref.quant(x[some]), ref.quant(w)
    with np.errstate(all="ignore"):
        v = (xc.astype(np.float64) @ wc.astype(np.float64).T) * xs[:, None].astype(np.float64) * ws.astype(np.float64)
        t = v + b
        # What float32 cannot hold is infinite before the activation.
        t = np.where(np.abs(t) < 2.0 ** 128, t, np.sign(t) * np.inf)
        want = ref.act(t, act, 0.25)
        grow, own = (1.13, 8) if act in (1, 4) else (1, 1)
        bound = U * (grow * (3 * np.abs(v) + np.abs(t)) + own * np.abs(t) + 2 * np.abs(want)) + 1e-37
    # Token 0 passes the range in channels 2 and 3, one each way.
    assert {t[0, 2], t[0, 3]} == {np.inf, -np.inf}
    odd = ~np.isfinite(t)
    assert rows == 1 or np.isnan(want[-1]).all()
    assert np.array_equal(got[some][odd], want[odd].astype(np.float32), equal_nan=True)
    assert np.all(np.abs(got[some][~odd] - want[~odd]) <= bound[~odd])
