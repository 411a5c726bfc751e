# SPDX-License-Identifier: Unlicense
"""CPU: norms with codes, the cache and attention within a window refuse bad
sizes, views beyond their buffers and overlaps on the host, before any launch;
sizes that are computed there, the binding's struct layouts. The addresses
below are never dereferenced."""

import ctypes as C

import pytest
from test_long_refusals import env, refused  # noqa: F401  (env is a fixture)


def test_sizes_and_layouts(ic):
    a = ic.api()
    assert [a.ops_cache_pitch(d) for d in (0, -1, 1, 16, 17, 100, 128, 129)] == [0, 0, 16, 16, 32, 112, 128, 0]
    for work in (a.ops_attention_window_work_bytes, a.ops_attention_cache_work_bytes):
        assert work(0, 4, 64) == work(4, 0, 64) == work(4, 4, 0) == work(4, 4, 129) == work(-1, 4, 64) == 0
        # Enough for every call of fewer rows, heads or channels; bounded.
        for d in (1, 32, 33, 64, 65, 128):
            sizes = [work(n, 4, d) for n in (1, 2, 31, 500, 513, 100000, 2 ** 31 - 1)]
            assert sizes == sorted(sizes) and sizes[0] > 0
            assert all(work(n, 4, d) <= work(n + 1, 4, d) <= work(n + 1, 5, d) <= work(n + 1, 5, min(128, d + 1))
                       for n in (1, 31, 127, 128, 500, 513, 100000))
        assert work(2 ** 31 - 1, 4096, 128) < 2 ** 27
    lib = ic.lib()
    assert C.sizeof(ic.Cache) == lib.icoreg_sizeof_cache()
    assert C.sizeof(ic.Seqs) == lib.icoreg_sizeof_seqs()


def test_norm(ic, env):  # noqa: F811
    a, o, v = env
    M = 1 << 20
    x, r, h, y, q, s, g = (v(i * M, M) for i in range(7))
    op = lambda b, off, ld: ic.Opnd(b, off, ld, 0, 0)  # noqa: E731
    none = op(None, 0, 0)

    def norm(rows=10, c=100, x=op(x, 0, 100), r=op(r, 0, 100), g=g, eps=1e-6, h=op(h, 0, 100), y=op(y, 0, 100), q=q, s=s):
        a.ops_rms_norm(o, rows, c, x, r, g, eps, h, y, q, s)

    for bad in (dict(rows=-1), dict(c=0), dict(rows=1 << 31), dict(c=(1 << 30) + 1)):
        with refused(ic, "ops_rms_norm: invalid sizes"):
            norm(**bad)
    for eps in (0.0, -1.0, float("nan"), float("inf")):
        with refused(ic, "ops_rms_norm: eps"):
            norm(eps=eps)
    xb, rb, hb = x, r, h
    for bad, match in ((dict(h=none, y=none, q=None, s=None), "no output"), (dict(q=None), "without"),
                       (dict(s=None), "without"), (dict(x=none), "X is NULL"),
                       (dict(x=op(xb, 0, 99)), "short row of X"), (dict(r=op(rb, -1, 100)), "short row of R"),
                       (dict(h=op(hb, 0, 99)), "short row of H"), (dict(y=op(y, 0, 99)), "short row of Y"),
                       (dict(x=op(xb, M // 4 - 999, 100)), "X accessed"), (dict(r=op(rb, M // 4 - 999, 100)), "R accessed"),
                       (dict(h=op(hb, M // 4 - 999, 100)), "H accessed"), (dict(y=op(y, M // 4 - 999, 100)), "Y accessed"),
                       (dict(g=v(0, 399)), "g accessed"), (dict(q=v(4 * M, 1279)), "Q accessed"),
                       (dict(s=v(5 * M, 39)), "S accessed"), (dict(q=v(4 * M + 8, M // 2)), "Q does not start"),
                       (dict(h=op(xb, 1, 100)), "H and an input"), (dict(y=op(rb, 4, 100)), "Y and an input"),
                       (dict(h=op(xb, 0, 101)), "H and an input"), (dict(y=op(hb, 50, 100)), "H and Y"),
                       (dict(y=op(hb, 0, 100)), "H and Y"), (dict(q=xb), "X and Q"), (dict(s=rb), "R and S"),
                       (dict(q=hb), "H and Q"), (dict(s=y), "Y and S"), (dict(s=q), "Q and S"), (dict(g=q), "g and Q"),
                       (dict(g=s), "g and S"), (dict(g=hb), "H and g")):
        with refused(ic, "ops_rms_norm: .*" + match):
            norm(**bad)
    norm(rows=0)


def parts(ic, v, M):
    """(cache, sequences) structs of sound views: 10 pages of 16 tokens of 2
    heads of 24 channels, 3 sequences of up to 4 pages."""
    cells = 10 * 2 * 16
    m = [v(20 * M + i * M, n) for i, n in enumerate((cells * 32, cells * 32, cells * 4, cells * 4, 16, 12, 48))]
    return ic.Cache(*m[:4], 10, 16, 2, 24), ic.Seqs(*m[4:], 3, 4), m


def changed(s, **kw):
    t = type(s)(*(getattr(s, n) for n, _ in s._fields_))
    for k, x in kw.items():
        setattr(t, k, x)
    return t


def cache_faults(ic, v, M, cache, seqs, m):
    """(cache, sequences, message) of what every call refuses."""
    for kw, match in ((dict(page=8), "page of 8"), (dict(page=48), "page of 48"), (dict(page=256), "page of 256"),
                      (dict(d=0), "head dimension 0"), (dict(d=129), "head dimension 129"), (dict(pages=-1), "invalid cache"),
                      (dict(nhk=0), "invalid cache"), (dict(pages=2 ** 31 - 1, nhk=2 ** 31 - 1), "invalid cache"),
                      (dict(kc=v(20 * M, 10239)), "kc accessed"), (dict(vc=None), "vc is NULL"),
                      (dict(ks=v(22 * M, 1279)), "ks accessed"), (dict(vs=v(23 * M, 1279)), "vs accessed"),
                      (dict(kc=v(20 * M + 8, M // 2)), "kc does not start"), (dict(vc=v(21 * M + 4, M // 2)), "vc does not start")):
        yield changed(cache, **kw), seqs, match
    for kw, match in ((dict(n=-1), "invalid sizes"), (dict(n=2 ** 31 - 1), "invalid sizes"), (dict(ldt=-1), "invalid sizes"),
                      (dict(ldt=2 ** 27), "invalid sizes"), (dict(start=v(24 * M, 15)), "start accessed"),
                      (dict(len=None), "len is NULL"), (dict(len=v(25 * M, 11)), "len accessed"),
                      (dict(table=v(26 * M, 47)), "table accessed")):
        yield cache, changed(seqs, **kw), match


def test_cache(ic, env):  # noqa: F811
    a, o, v = env
    M = 1 << 20
    cache, seqs, m = parts(ic, v, M)
    K, V = v(0, M), v(M, M)
    op = lambda b, off=0, ld=48: ic.Opnd(b, off, ld, 0, 0)  # noqa: E731
    for name, call in (("ops_cache_write", a.ops_cache_write), ("ops_cache_read", a.ops_cache_read)):
        def move(c=cache, s=seqs, rows=20, k=op(K), x=op(V)):
            call(o, C.byref(c), C.byref(s), rows, k, x)

        for c, s, match in cache_faults(ic, v, M, cache, seqs, m):
            with refused(ic, f"{name}: .*{match}"):
                move(c, s)
        faults = [(dict(rows=-1), "invalid sizes"), (dict(k=op(K, 0, 47)), "short row of K"),
                  (dict(x=op(V, -1)), "short row of V"), (dict(k=op(K, M // 4 - 959)), "K accessed"),
                  (dict(x=op(V, M // 4 - 959)), "V accessed"), (dict(k=op(m[0])), "K and kc"), (dict(x=op(m[3], 0)), "V accessed|V and vs"),
                  (dict(c=changed(cache, vc=m[0])), "kc and vc"), (dict(c=changed(cache, ks=m[1])), "vc and ks"),
                  (dict(c=changed(cache, vs=m[2])), "ks and vs"), (dict(s=changed(seqs, table=m[2])), "the cache and table"),
                  (dict(s=changed(seqs, start=m[0])), "the cache and start"), (dict(s=changed(seqs, len=m[3])), "the cache and len")]
        if name == "ops_cache_write":
            faults += [(dict(k=op(None)), "has no buffer"), (dict(x=op(None)), "has no buffer")]
        else:
            faults += [(dict(k=op(None), x=op(None)), "has no buffer"), (dict(x=op(K, 20)), "K and V"),
                       (dict(s=changed(seqs, start=K)), "K and start"), (dict(s=changed(seqs, table=V)), "V and table")]
        for bad, match in faults:
            with refused(ic, f"{name}: .*({match})"):
                move(**bad)
        with refused(ic, f"{name}: no cache or no sequences"):
            call(o, None, C.byref(seqs), 20, op(K), op(V))
        with refused(ic, f"{name}: no cache or no sequences"):
            call(o, C.byref(cache), None, 20, op(K), op(V))
        # Nothing to do.
        move(rows=0, k=op(None), x=op(None))
        move(s=changed(seqs, n=0, start=None, len=None, table=None))
        with refused(ic, f"{name}: 16777216 blocks of 512 threads exceed a launch|{name}: .* exceed a launch"):
            huge = [ic.lib().ocl_wrap(C.c_void_p((i + 1) << 45), 1 << 43) for i in range(2)]
            move(changed(cache, d=24), rows=2 ** 31 - 1, k=op(huge[0]), x=op(huge[1]))
        for h in huge:
            ic.lib().ocl_release(C.byref(h))


def test_window(ic, env):  # noqa: F811
    a, o, v = env
    M = 1 << 22
    q, k, val, out, mask, work = (v(i * M, M) for i in range(6))
    work = v(5 * M, 8 * M)
    kb, vb, qb, ob, wb = k, val, q, out, work
    op = lambda b, off, ld: ic.Opnd(b, off, ld, 0, 0)  # noqa: E731
    need = a.ops_attention_window_work_bytes(20, 4, 32)

    def window(q=op(q, 0, 128), k=op(k, 0, 64), val=op(val, 0, 64), out=op(out, 0, 128), nq=20, nk=100, h=4, kv=2, d=32, q0=0,
               left=5, right=5, sinks=1, mask=mask, work=work):
        a.ops_attention_window(o, q, k, val, out, nq, nk, h, kv, d, q0, left, right, sinks, 0.2, mask, work)

    for bad, match in ((dict(d=0), "head dimension 0"), (dict(d=129), "head dimension 129"), (dict(nq=-1), "invalid sizes"),
                       (dict(nk=-1), "invalid sizes"), (dict(nk=2 ** 31 - 1), "invalid sizes"), (dict(h=0), "invalid sizes"),
                       (dict(kv=0), "invalid sizes"), (dict(kv=3), "invalid sizes"), (dict(sinks=-1), "invalid sizes"),
                       (dict(q0=2 ** 31 - 1), "invalid sizes"), (dict(q0=-2 ** 31), "invalid sizes"),
                       (dict(q=op(qb, 0, 127)), "short row"), (dict(out=op(ob, -1, 128)), "short row"),
                       (dict(k=op(kb, 0, 63)), "short row of K or V"), (dict(val=op(vb, -1, 64)), "short row of K or V"),
                       (dict(q=op(qb, M // 4 - 2559, 128)), "Q accessed"), (dict(out=op(ob, M // 4 - 2559, 128)), "O accessed"),
                       (dict(k=op(kb, M // 4 - 6399, 64)), "K accessed"), (dict(val=op(vb, M // 4 - 6399, 64)), "V accessed"),
                       (dict(mask=v(0, 99)), "kmask accessed"), (dict(work=v(5 * M, need - 1)), "work accessed"),
                       (dict(work=None), "work is NULL"), (dict(work=v(5 * M + 8, 2 * M)), "work does not start"),
                       (dict(out=op(qb, 4, 128)), "O and Q"), (dict(out=op(kb, 0, 128)), "O and K"),
                       (dict(out=op(vb, 0, 128)), "O and V"), (dict(mask=ob), "kmask and O"), (dict(out=op(wb, 0, 128)), "O and work"),
                       (dict(q=op(wb, 0, 128)), "Q and work"), (dict(k=op(wb, 0, 64)), "K and work"),
                       (dict(val=op(wb, 0, 64)), "V and work"), (dict(mask=wb), "kmask and work")):
        with refused(ic, "ops_attention_window: .*" + match):
            window(**bad)
    window(nq=0, work=None)


def test_attention_cache(ic, env):  # noqa: F811
    a, o, v = env
    M = 1 << 20
    cache, seqs, m = parts(ic, v, M)
    q, out, work = v(0, M), v(M, M), v(2 * M, 8 * M)
    op = lambda b, off=0, ld=96: ic.Opnd(b, off, ld, 0, 0)  # noqa: E731
    need = a.ops_attention_cache_work_bytes(20, 4, 24)
    qb, ob = q, out

    def attend(c=cache, s=seqs, rows=20, q=op(q), out=op(out), h=4, left=-1, sinks=0, work=work):
        a.ops_attention_cache(o, C.byref(c), C.byref(s), rows, q, out, h, left, sinks, 0.2, work)

    for c, s, match in cache_faults(ic, v, M, cache, seqs, m):
        with refused(ic, f"ops_attention_cache: .*{match}"):
            attend(c, s)
    for bad, match in ((dict(rows=-1), "invalid sizes"), (dict(h=3), "invalid sizes"), (dict(h=0), "invalid sizes"),
                       (dict(sinks=-1), "invalid sizes"), (dict(q=op(qb, 0, 95)), "short row"), (dict(out=op(ob, -1)), "short row"),
                       (dict(q=op(qb, M // 4 - 1919)), "Q accessed"), (dict(out=op(ob, M // 4 - 1919)), "O accessed"),
                       (dict(work=v(2 * M, need - 1)), "work accessed"), (dict(work=v(2 * M + 8, M)), "work does not start|work accessed"),
                       (dict(out=op(qb, 4)), "O and Q"), (dict(out=op(work)), "O and work"), (dict(q=op(work)), "Q and work"),
                       (dict(out=op(m[0], 0, 96), c=changed(cache, kc=v(20 * M, M))), "O accessed|O and kc"),
                       (dict(s=changed(seqs, table=ob)), "O and table"), (dict(s=changed(seqs, start=work)), "work and start"),
                       (dict(c=changed(cache, vc=work)), "work and vc")):
        with refused(ic, f"ops_attention_cache: .*({match})"):
            attend(**bad)
    attend(rows=0, work=None)
    attend(s=changed(seqs, n=0, start=None, len=None, table=None), work=None)
