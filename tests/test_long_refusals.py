# SPDX-License-Identifier: Unlicense
"""CPU: the operators for long sequences refuse bad sizes, views beyond their
buffers and overlaps on the host, before any launch; frequencies and sizes
that are computed there. The addresses below are never dereferenced."""

import ctypes as C

import numpy as np
import pytest

BASE = 1 << 24


@pytest.fixture
def env(ic):
    """(checked api, ops, a maker of views at byte offsets of one place)."""
    lib, be, o, made = ic.lib(), ic.OclBackend(cu_count=256), ic.Ops(), []
    o.ocl = C.pointer(be)

    def view(off, n):
        made.append(lib.ocl_wrap(C.c_void_p(BASE + off), n))
        return made[-1]
    yield ic.api(), C.byref(o), view
    for m in made:
        lib.ocl_release(C.byref(m))


def refused(ic, match):
    return pytest.raises(ic.IcoregError, match=match)


def test_sizes(ic):
    a = ic.api()
    assert [a.ops_q8_pitch(c) for c in (0, -1, 1, 64, 65, 4096)] == [0, 0, 64, 64, 128, 4096]
    assert a.ops_linear_q8_work_bytes(3, 65) >= 3 * 128 + 12
    assert a.ops_linear_q8_work_bytes(0, 65) == a.ops_linear_q8_work_bytes(3, (1 << 17) + 1) == 0
    assert [a.ops_key_blocks(n, b) for n, b in ((0, 16), (1, 16), (16, 16), (17, 16), (2 ** 31 - 1, 64), (5, 48))] == \
        [0, 1, 1, 2, 0, 0]
    assert a.ops_attention_blocks_work_bytes(5, 100, 4, 2, 64, 32, 3) >= 5 * 4 * 3 * 64 * 4
    for bad in ((5, 100, 4, 3, 64, 32, 3), (5, 100, 4, 2, 129, 32, 3), (5, 100, 4, 2, 64, 33, 3),
                (5, 100, 4, 2, 64, 32, 65), (-1, 100, 4, 2, 64, 32, 3), (0, 100, 4, 2, 64, 32, 3)):
        assert a.ops_attention_blocks_work_bytes(*bad) == 0


def test_work_stays_bounded(ic):
    """Long batches are computed in passes: the work of a hundred times the
    queries is not a hundred times the work."""
    a = ic.api()
    one, many = (a.ops_attention_blocks_work_bytes(n, 65536, 16, 16, 128, 64, 16) for n in (8192, 819200))
    assert one <= many < 2 ** 31


def test_quant_rows(ic, env):
    a, o, v = env
    x, q, s = v(0, 4000), v(8192, 2560), v(16384, 40)
    for sizes in ((-1, 100, 100), (10, 0, 100), (10, 100, 99), (1 << 31, 1, 1),
                  (1, (1 << 30) + 1, 1 << 31 - 1)):
        with refused(ic, "ops_quant_rows: invalid sizes"):
            a.ops_quant_rows(o, sizes[0], sizes[1], x, 0, sizes[2], q, s)
    with refused(ic, "ops_quant_rows: X accessed"):
        a.ops_quant_rows(o, 10, 100, x, 1, 100, q, s)
    with refused(ic, "ops_quant_rows: Q accessed"):
        a.ops_quant_rows(o, 10, 100, x, 0, 100, v(8192, 1279), s)
    with refused(ic, "ops_quant_rows: S accessed"):
        a.ops_quant_rows(o, 10, 100, x, 0, 100, q, v(16384, 39))
    with refused(ic, "ops_quant_rows: S is NULL"):
        a.ops_quant_rows(o, 10, 100, x, 0, 100, q, None)
    with refused(ic, "Q does not start on a multiple of 16"):
        a.ops_quant_rows(o, 10, 100, x, 0, 100, v(8200, 2560), s)
    with refused(ic, "X and Q must not overlap"):
        a.ops_quant_rows(o, 10, 100, x, 0, 100, v(3984, 2560), s)
    with refused(ic, "S and X must not overlap"):
        a.ops_quant_rows(o, 10, 100, x, 0, 100, q, v(3996, 40))
    with refused(ic, "S and Q must not overlap"):
        a.ops_quant_rows(o, 10, 100, x, 0, 100, q, v(8192 + 1276, 40))
    a.ops_quant_rows(o, 0, 100, None, 0, 100, None, None)


def test_linear(ic, env):
    a, o, v = env
    M = 1 << 20
    rows, cin, cout = 8, 100, 30
    x, wq, ws, b, y, work = v(0, M), v(M, 30 * 128), v(2 * M, 120), v(3 * M, 120), v(4 * M, M), v(6 * M, M)

    def q8(rows=rows, cin=cin, cout=cout, x=x, xoff=0, ldx=cin, wq=wq, ws=ws, b=b, r=None, roff=0, y=y, yoff=0,
           ldy=cout, act=0, work=work):
        a.ops_linear_q8(o, rows, cin, cout, x, xoff, ldx, wq, ws, b, r, roff, y, yoff, ldy, act, 0.0, work)

    for bad in (dict(rows=-1), dict(cin=0), dict(cin=(1 << 17) + 1, ldx=1 << 18), dict(cout=-1), dict(ldy=29),
                dict(yoff=-1), dict(roff=-1), dict(ldx=99), dict(xoff=-1)):
        with refused(ic, "ops_linear_q8: invalid sizes"):
            q8(**bad)
    # Tokens and channels are counted past the last.
    for bad in (dict(rows=2 ** 31 - 1), dict(cout=2 ** 31 - 1, ldy=2 ** 31 - 1)):
        with refused(ic, "ops_linear_q8: invalid sizes"):
            q8(**bad)
    assert a.ops_linear_q8_work_bytes(2 ** 31 - 1, 64) == 0
    with refused(ic, "invalid activation 5"):
        q8(act=5)
    for bad, name in ((dict(xoff=M // 4 - 799), "X"), (dict(wq=v(M, 3839)), "WQ"), (dict(ws=v(2 * M, 119)), "WS"),
                      (dict(b=v(3 * M, 119)), "bias"), (dict(yoff=M // 4 - 239), "Y"),
                      (dict(r=v(5 * M, 959)), "R"), (dict(work=v(6 * M, 1055)), "work")):
        with refused(ic, f"ops_linear_q8: {name} accessed"):
            q8(**bad)
    with refused(ic, "WQ does not start"):
        q8(wq=v(M + 4, 30 * 128))
    with refused(ic, "work does not start"):
        q8(work=v(6 * M + 8, M))
    for bad, names in ((dict(y=x), "Y and X"), (dict(y=wq, wq=wq), "Y and WQ"), (dict(work=y), "Y and work"),
                       (dict(work=x), "X and work"), (dict(r=y, roff=1), "Y and R"),
                       (dict(y=v(2 * M, M)), "Y and WS"), (dict(y=v(3 * M, M)), "Y and bias"),
                       (dict(work=v(M, M)), "WQ and work"), (dict(work=v(2 * M, M)), "WS and work"),
                       (dict(work=v(3 * M, M)), "bias and work"), (dict(r=work), "R and work")):
        with refused(ic, names):
            q8(**bad)
    q8(rows=0)
    q8(cout=0, ldy=0)
    xq, xs = v(7 * M, 1024), v(8 * M, 32)

    def qq(xq=xq, xs=xs, y=y):
        a.ops_linear_qq(o, rows, cin, cout, xq, xs, wq, ws, b, None, 0, y, 0, cout, 0, 0.0)

    for bad, match in ((dict(xq=v(7 * M, 1023)), "XQ accessed"), (dict(xs=v(8 * M, 31)), "XS accessed"),
                       (dict(xq=v(7 * M + 1, 2048)), "XQ does not start"), (dict(y=v(7 * M + 1000, M)), "Y and XQ"),
                       (dict(y=v(8 * M + 16, M)), "Y and XS")):
        with refused(ic, "ops_linear_qq: " + match):
            qq(**bad)


def test_rope(ic, env):
    a, o, v = env
    M = 1 << 20
    x, y, z, pos, freq = v(0, M), v(M, M), v(2 * M, M), v(3 * M, 40), v(4 * M, 64)
    op = lambda b, off, ld: ic.Opnd(b, off, ld, 0, 0)  # noqa: E731

    def rope(rows=10, d=16, rot=16, axes=1, pos=pos, freq=freq, flags=0, x1=op(x, 0, 64), y1=op(y, 0, 64), n1=4,
             x2=op(None, 0, 0), y2=op(None, 0, 0), n2=0):
        a.ops_rope_pos(o, rows, d, rot, axes, pos, freq, 1.0, flags, x1, y1, n1, x2, y2, n2)

    for bad in (dict(rows=-1), dict(d=0), dict(rot=3), dict(rot=-2), dict(rot=18), dict(axes=0), dict(axes=5),
                dict(n1=-1), dict(n2=-1), dict(flags=4), dict(d=4000, rot=2050)):
        with refused(ic, "ops_rope_pos: invalid sizes"):
            rope(**bad)
    for bad in (dict(x1=op(x, 0, 63)), dict(y1=op(y, 0, 63)), dict(x1=op(x, -1, 64)), dict(y1=op(y, -1, 64))):
        with refused(ic, "invalid sizes of X1 or Y1"):
            rope(**bad)
    with refused(ic, "X1 or Y1 accessed"):
        rope(x1=op(x, M // 4 - 639, 64))
    with refused(ic, "X2 or Y2 is NULL"):
        rope(n2=1, x2=op(None, 0, 16), y2=op(z, 0, 16))
    with refused(ic, "pos accessed"):
        rope(axes=2)
    with refused(ic, "freq accessed"):
        rope(freq=v(4 * M, 63))
    with refused(ic, "freq does not start"):
        rope(freq=v(4 * M + 4, 64))
    with refused(ic, "an output and an input"):
        rope(y1=op(x, 1, 64))
    with refused(ic, "an output and an input"):
        rope(y1=op(x, 0, 80))
    with refused(ic, "an output and an input"):
        # Keys over the queries' inputs.
        rope(n2=1, x2=op(z, 0, 16), y2=op(x, 48, 64))
    for bad, match in ((dict(y1=op(pos, 0, 64), rows=1, n1=1, d=8, rot=8, x1=op(x, 0, 64)), "an output and pos"),
                       (dict(y1=op(freq, 0, 64), rows=1, n1=1, d=8, rot=8, x1=op(x, 0, 64)), "an output and freq")):
        with refused(ic, match):
            rope(**bad)
    with refused(ic, "Y1 and Y2"):
        rope(n2=1, x2=op(z, 0, 16), y2=op(y, 63, 64))
    rope(rows=0)
    rope(n1=0)


def test_frequencies(ic):
    a = ic.api()

    def freqs(rot, axes=1, base=10000.0, kind=0, factor=1.0, trained=0.0, slow=0.0, fast=0.0):
        f = np.full(rot // 2, -1.0)
        a.ops_rope_freqs(f.ctypes.data, rot, axes, base, kind, factor, trained, slow, fast)
        return f

    k = np.arange(32)
    w = 10000.0 ** (-2 * k / 64)
    assert np.allclose(freqs(64), w, rtol=1e-14)
    assert np.allclose(freqs(64, kind=1, factor=4.0), w / 4, rtol=1e-14)
    assert np.allclose(freqs(64, 2), 10000.0 ** (-2 * (k // 2) / 32), rtol=1e-14)
    # Another base: the fastest pair stays, the slowest is stretched by factor.
    f = freqs(64, kind=2, factor=4.0)
    assert f[0] == 1 and np.isclose(f[-1], w[-1] / 4, rtol=1e-13)
    f = freqs(64, kind=3, factor=16.0, trained=4096.0, slow=1.0, fast=32.0)
    turns = 4096 * w / (2 * np.pi)
    assert np.allclose(f[turns >= 32], w[turns >= 32], rtol=1e-14)
    assert np.allclose(f[turns <= 1], w[turns <= 1] / 16, rtol=1e-14)
    g = (turns - 1) / 31
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and np.allclose(f[mid], (w * (g + (1 - g) / 16))[mid], rtol=1e-13)
    assert freqs(2, kind=2, factor=4.0)[0] == 1
    for bad in (dict(rot=64, axes=0), dict(rot=62, axes=2), dict(rot=64, kind=4), dict(rot=64, base=0.0),
                dict(rot=64, factor=0.0), dict(rot=64, factor=float("nan"))):
        with refused(ic, "ops_rope_freqs: invalid arguments"):
            freqs(**bad)
    with refused(ic, "ops_rope_freqs: invalid range"):
        freqs(64, kind=3, trained=4096.0, slow=2.0, fast=2.0)


def test_blocks(ic, env):
    a, o, v = env
    M = 1 << 22
    q, k, val, out, kc, ks, sel, mask, work = (v(i * M, M) for i in range(9))
    kb, vb, qb, ob = k, val, q, out
    op = lambda b, off, ld: ic.Opnd(b, off, ld, 0, 0)  # noqa: E731
    nq, nk, h, kv, d, bs, top = 20, 100, 4, 2, 32, 16, 3

    def index(k=op(k, 0, 64), nk=nk, kv=kv, d=d, bs=bs, mask=mask, b0=0, nb=7, kc=kc, ks=ks):
        a.ops_block_index(o, k, nk, kv, d, bs, mask, b0, nb, kc, ks)

    for bad, match in ((dict(bs=48), "block size 48"), (dict(d=129), "head dimension 129"), (dict(d=0), "head dim"),
                       (dict(nk=-1, nb=0), "invalid sizes"), (dict(kv=0), "invalid sizes"),
                       (dict(b0=-1), "invalid sizes"), (dict(nb=8), "invalid sizes"), (dict(nb=-1), "invalid sizes"),
                       (dict(b0=7, nb=1), "invalid sizes"), (dict(k=op(k, 0, 63)), "invalid sizes"),
                       (dict(k=op(k, -1, 64)), "invalid sizes"), (dict(k=op(k, M // 4 - 6399, 64)), "K accessed"),
                       (dict(mask=v(0, 99)), "kmask accessed"), (dict(kc=v(0, 14 * 64 - 1)), "KC accessed"),
                       (dict(ks=v(0, 14 * 4 - 1)), "KS accessed"), (dict(kc=v(8, M)), "KC does not start"),
                       (dict(nk=2 ** 31 - 1, nb=0), "invalid sizes"), (dict(kc=kb), "KC and K"),
                       (dict(ks=kb), "KS and K"), (dict(ks=kc), "KC and KS"), (dict(mask=kc), "KC and kmask"),
                       (dict(mask=ks), "KS and kmask")):
        with refused(ic, "ops_block_index: .*" + match):
            index(**bad)
    index(nb=0)

    def select(q=op(q, 0, 128), nq=nq, h=h, kv=kv, d=d, kc=kc, ks=ks, n=7, top=top, sel=sel, work=work):
        a.ops_block_select(o, q, nq, h, kv, d, kc, ks, n, top, sel, work)

    for bad, match in ((dict(d=129), "head dimension"), (dict(top=0), "0 blocks"), (dict(top=65), "65 blocks"),
                       (dict(kv=3), "invalid sizes"), (dict(h=0), "invalid sizes"), (dict(nq=-1), "invalid sizes"),
                       (dict(n=-1), "invalid sizes"), (dict(n=2 ** 27 + 1), "invalid sizes"),
                       (dict(q=op(q, 0, 127)), "invalid sizes"),
                       (dict(q=op(q, M // 4 - 2559, 128)), "Q accessed"), (dict(kc=v(0, 14 * 64 - 1)), "KC accessed"),
                       (dict(ks=None), "KS is NULL"), (dict(sel=v(0, 959)), "SEL accessed"),
                       (dict(kc=v(8, M)), "KC does not start"), (dict(sel=qb), "SEL and Q"),
                       (dict(sel=kc), "SEL and KC"), (dict(sel=ks), "SEL and KS")):
        with refused(ic, "ops_block_select: .*" + match):
            select(**bad)
    select(nq=0)

    def attend(q=op(q, 0, 128), k=op(k, 0, 64), val=op(val, 0, 64), out=op(out, 0, 128), nq=nq, nk=nk, h=h, kv=kv,
               d=d, bs=bs, top=top, sel=sel, mask=mask, work=work):
        a.ops_attention_blocks(o, q, k, val, out, nq, nk, h, kv, d, bs, top, sel, 0.2, mask, work)

    for bad, match in ((dict(d=129), "invalid sizes"), (dict(bs=8), "invalid sizes"), (dict(top=65), "invalid sizes"),
                       (dict(kv=3), "invalid sizes"), (dict(nk=-1), "invalid sizes"), (dict(nq=-1), "invalid sizes"),
                       (dict(q=op(qb, 0, 127)), "short row"), (dict(val=op(vb, 0, 63)), "short row"),
                       (dict(out=op(ob, -1, 128)), "negative offset"), (dict(q=op(qb, M // 4 - 2559, 128)), "Q accessed"),
                       (dict(k=op(kb, M // 4 - 6399, 64)), "K accessed"),
                       (dict(val=op(vb, M // 4 - 6399, 64)), "V accessed"),
                       (dict(out=op(ob, M // 4 - 2559, 128)), "O accessed"), (dict(sel=v(0, 959)), "SEL accessed"),
                       (dict(mask=v(0, 99)), "kmask accessed"), (dict(work=v(8 * M, 63)), "work accessed"),
                       (dict(work=None), "work is NULL"), (dict(work=v(8 * M + 4, M)), "work does not start"),
                       (dict(out=op(qb, 4, 128)), "O and Q"), (dict(out=op(kb, 0, 128)), "O and K"),
                       (dict(out=op(vb, 0, 128)), "O and V"), (dict(work=ob), "O and work"),
                       (dict(work=sel), "SEL and work"), (dict(sel=ob), "SEL and O"), (dict(mask=ob), "kmask and O"),
                       (dict(work=qb), "Q and work"), (dict(work=kb), "K and work"), (dict(work=vb), "V and work"),
                       (dict(work=mask), "kmask and work")):
        with refused(ic, "ops_attention_blocks: .*" + match):
            attend(**bad)
    attend(nq=0)


def test_launches(ic, env):
    """More blocks of threads than a launch takes are refused by name, and
    units too many for the 32-bit places of the lists go one by one."""
    a, o, _ = env
    huge = [ic.lib().ocl_wrap(C.c_void_p((i + 1) << 44), 1 << 43) for i in range(4)]
    op = lambda b, ld: ic.Opnd(b, 0, ld, 0, 0)  # noqa: E731
    with refused(ic, "selection rows: 67108864 blocks of 64 threads exceed a launch"):
        a.ops_block_select(o, op(huge[0], 1), 1 << 26, 1, 1, 1, huge[1], huge[2], 600, 1, huge[3], None)
    with refused(ic, "block index: 16777216 blocks of 256 threads exceed a launch"):
        a.ops_block_index(o, op(huge[0], 16), 1 << 24, 16, 1, 16, None, 0, 1 << 20, huge[1], huge[2])
    # A row in several units of 2048 channels.
    with refused(ic, "rope blocks: 16777216 blocks of 256 threads exceed a launch"):
        a.ops_rope_pos(o, 1 << 24, 2048, 2048, 1, huge[2], huge[3], 1.0, 0, op(huge[0], 2048), op(huge[0], 2048), 1,
                       op(None, 0), op(None, 0), 0)
    for m in huge:
        ic.lib().ocl_release(C.byref(m))
    choose = ic.lib().icoreg_blocks_choice
    assert choose(1, 2048, 65536, 1, 128, 64, 64) == 1
    assert choose(1, 2048, 131072, 1, 128, 64, 64) == 1
    assert choose(1, 2048, 131073, 1, 128, 64, 64) == 0


# Heads, key heads, channels, block, top.
WORK = [(8, 2, 64, 64, 16), (16, 16, 128, 64, 16), (4, 1, 32, 16, 1), (1, 1, 16, 128, 64), (12, 4, 100, 32, 7),
        (16, 4, 128, 64, 16), (65540, 65540, 8, 16, 2)]


@pytest.mark.parametrize("h,kv,d,bs,top", WORK)
def test_work_covers_every_shorter_call(h, kv, d, bs, top, ic):
    """The work of a call is enough for every call of fewer queries or keys:
    across the border where one pass becomes two, and where units go by
    lists, one by one otherwise."""
    work = ic.api().ops_attention_blocks_work_bytes
    rng = np.random.default_rng(h + d)
    one = [work(n, 100, h, kv, d, bs, top) for n in (1, 2)]
    border = (512 << 20) // max(1, one[1] - one[0])
    queries = sorted({1, 2, 3, 64, *(max(1, m * border + e) for m in (1, 2, 3) for e in (-2, -1, 0, 1, 2)),
                      *(int(x) for x in np.exp(rng.uniform(0, np.log(3 * border + 64), 40)))})
    keys = sorted({0, 1, 16380, 52416, 52480, *(int(x) for x in np.exp(rng.uniform(0, np.log(4e6), 60)))})
    size = np.array([[work(n, k, h, kv, d, bs, top) for k in keys] for n in queries])
    used, passes, n = np.zeros_like(size), set(), C.c_size_t()
    for i, nq in enumerate(queries):
        for j, nk in enumerate(keys):
            passes.add(ic.lib().icoreg_blocks_passes(nq, nk, h, kv, d, bs, top, C.byref(n)))
            used[i, j] = n.value
    assert (used <= size).all() and {1, 2, 3} <= passes
    assert (np.diff(size, axis=0) >= 0).all() and (np.diff(size, axis=1) >= 0).all()
    # By the number of blocks listed, too.
    for n, k in ((1, 5000), (700, 5000), (border, 5000), (3 * border, 5000)):
        assert (np.diff([work(n, k, h, kv, d, bs, t) for t in range(1, 65)]) >= 0).all()
