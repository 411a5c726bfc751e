# SPDX-License-Identifier: Unlicense
"""GPU: norms with codes, the cache and attention within a window as a
transformer layer uses them: the norm's codes into a packed projection of
queries, keys and values, rotary positions in place, keys and values into the
cache, attention over it, the output projection, and the norm that adds it to
the residual; prompts of several sequences in one pass, then single tokens of
all of them from one recording.

Every step is held to its own definition on the inputs that it was given, so
that a rounding that moves a code in one of them is not an error of the next."""

import numpy as np
import pytest

import kept_ref
import long_ref as ref
import test_q8_gpu as q8
from kept_ref import sees
from long_ref import U
from test_cache_gpu import Held
from test_window_gpu import check, run

pytestmark = pytest.mark.gpu

C, H, KV, D, PAGE, EPS = 256, 8, 2, 32, 32, 1e-5
W, WK = H * D, KV * D
WIDE = W + 2 * WK


class Layer:
    def __init__(self, dev, ic, n, most, left, sinks):
        self.dev, self.ic, self.left, self.sinks = dev, ic, left, sinks
        rng = np.random.default_rng(n)
        self.wqkv = (rng.standard_normal((WIDE, C)) * 1.5 / C ** 0.5).astype(np.float32)
        self.wo = (rng.standard_normal((C, W)) / W ** 0.5).astype(np.float32)
        self.g = [(1 + 0.3 * rng.standard_normal(C)).astype(np.float32) for _ in "ab"]
        self.freq = np.zeros(D // 2)
        ic.api().ops_rope_freqs(self.freq.ctypes.data, D, 1, 10000.0, 0, 1.0, 0.0, 0.0, 0.0)
        self.weights = [self._weight(w) for w in (self.wqkv, self.wo)]
        self.F, self.G = dev.upload(self.freq), [dev.upload(g) for g in self.g]
        self.held = Held(dev, ic, 60, PAGE, KV, D)
        a, f = dev.api, dev.zeros
        self.X, self.QKV, self.O, self.Y, self.H = f(most * C), f(most * WIDE), f(most * W), f(most * C), f(most * C)
        self.P = f(most, np.int32)
        self.codes = [(dev.alloc(most * ref.pitch(C)), f(most)) for _ in "ab"]
        self.work = dev.alloc(max(a.ops_linear_q8_work_bytes(most, W), a.ops_attention_cache_work_bytes(most, H, D)))

    def _weight(self, w):
        dev = self.dev
        M, Q, S = dev.upload(w), dev.alloc(len(w) * ref.pitch(w.shape[1])), dev.alloc(len(w) * 4)
        dev.api.ops_quant_rows(dev.po, *w.shape, M.mem, 0, w.shape[1], Q.mem, S.mem)
        return Q, S

    def launch(self, s, rows):
        dev, ic, a = self.dev, self.ic, self.dev.api
        none, m = ic.Opnd(None, 0, 0, 0, 0), lambda o: ic.mat(self.QKV, o, WIDE)  # noqa: E731
        x, y, h = (ic.mat(b, 0, C) for b in (self.X, self.Y, self.H))
        (q1, s1), (q2, s2) = self.codes
        (wq, ws), (oq, os) = self.weights
        a.ops_rms_norm(dev.po, rows, C, x, none, self.G[0].mem, EPS, none, none, q1.mem, s1.mem)
        a.ops_linear_qq(dev.po, rows, C, WIDE, q1.mem, s1.mem, wq.mem, ws.mem, None, None, 0, self.QKV.mem, 0, WIDE, 0, 0.0)
        a.ops_rope_pos(dev.po, rows, D, D, 1, self.P.mem, self.F.mem, 1.0, 1, m(0), m(0), H, m(W), m(W), KV)
        a.ops_cache_write(dev.po, self.held.p, ic.C.byref(s), rows, m(W), m(W + WK))
        a.ops_attention_cache(dev.po, self.held.p, ic.C.byref(s), rows, m(0), ic.mat(self.O, 0, W), H, self.left, self.sinks,
                              float(np.float32(D ** -0.5)), self.work.mem)
        a.ops_linear_q8(dev.po, rows, W, C, self.O.mem, 0, W, oq.mem, os.mem, None, None, 0, self.Y.mem, 0, C, 0, 0.0,
                        self.work.mem)
        a.ops_rms_norm(dev.po, rows, C, x, y, self.G[1].mem, EPS, h, y, q2.mem, s2.mem)

    def codes_of(self, i, n):
        q, s = self.codes[i]
        return self.dev.read(q, n * ref.pitch(C), np.int8).reshape(n, -1)[:, :C], self.dev.read(s, n)

    def checked(self, x, start, lengths, table):
        """What launch left, of rows x."""
        dev, n, scale = self.dev, len(x), np.float32(D ** -0.5)
        _, y1 = kept_ref.rms_norm(x, None, self.g[0], np.float32(EPS))
        for got, want in zip(self.codes_of(0, n), ref.quant(y1)):
            assert np.array_equal(got, want)
        qkv = dev.read(self.QKV, n * WIDE).reshape(n, WIDE)
        want, bound = q8.expected(y1, self.wqkv, None, None, 0, 0)
        # Values as they were projected, queries and keys turned: a rotation
        # keeps a pair's error to its length, sqrt(2) of either's at most.
        assert np.all(np.abs(qkv - want)[:, W + WK:] <= bound[:, W + WK:])
        pos = np.concatenate([np.arange(lengths[b] - (start[b + 1] - start[b]), lengths[b]) for b in range(len(lengths))])
        heads = want[:, :W + WK].reshape(n, H + KV, D)
        turned = ref.rope(heads, pos[:, None], self.freq, D, True)
        most = 2 * bound[:, :W + WK].reshape(n, H + KV, D).max(-1, keepdims=True) + 12 * U * np.abs(heads).max()
        assert np.all(np.abs(qkv[:, :W + WK].reshape(n, H + KV, D) - turned) <= most)
        q, k, v = (qkv[:, o:o + m * D].reshape(n, m, D) for o, m in ((0, H), (W, KV), (W + WK, KV)))
        self.held.ref.write(k, v, start, lengths, table)
        self.held.matches()
        o = dev.read(self.O, n * W).reshape(n, H, D)
        for b in range(len(lengths)):
            at = slice(start[b], start[b + 1])
            k8, v8, kept = self.held.ref.keys(b, lengths, table)
            check(o[at], q[at], k8, v8, sees(pos[at], len(k8), self.left, 0, self.sinks) & kept, scale)
        h, y = dev.read(self.H, n * C).reshape(n, C), dev.read(self.Y, n * C).reshape(n, C)
        want, bound = q8.expected(o.reshape(n, W), self.wo, None, None, 0, 0)
        assert np.all(np.abs(h.astype(np.float64) - x - want) <= bound + U * np.abs(h))
        _, y2 = kept_ref.rms_norm(h, None, self.g[1], np.float32(EPS))
        assert np.array_equal(y, y2)
        for got, want in zip(self.codes_of(1, n), ref.quant(y2)):
            assert np.array_equal(got, want)
        return q, o


@pytest.mark.parametrize("prompts,left,sinks", [([5], -1, 0), ([100, 31, 64], -1, 0), ([200, 1, 90], 50, 4)])
def test_prompts_then_tokens(prompts, left, sinks, dev, ic):
    print(f"[kept layer] {prompts}: {left} {sinks}", flush=True)
    n, total = len(prompts), sum(prompts)
    rng = np.random.default_rng(total)
    layer = Layer(dev, ic, n, total, left, sinks)
    lengths, start = np.array(prompts, np.int32), np.concatenate([[0], np.cumsum(prompts)])
    table = rng.permutation(60)[:n * 12].reshape(n, 12).astype(np.int32)
    x = rng.standard_normal((total, C)).astype(np.float32)
    dev.write(layer.X, x)
    dev.write(layer.P, np.concatenate([np.arange(m) for m in prompts]).astype(np.int32))
    layer.launch(layer.held.seqs(start, lengths, table), total)
    q, o = layer.checked(x, start, lengths, table)
    # The kept keys and values read back, and the same attention over them.
    b = int(np.argmax(prompts))
    m = prompts[b]
    one = layer.held.seqs([0, m], [m], table[b:b + 1])
    K, V = dev.zeros(m * WK), dev.zeros(m * WK)
    dev.api.ops_cache_read(dev.po, layer.held.p, ic.C.byref(one), m, ic.mat(K, 0, WK), ic.mat(V, 0, WK))
    k, v = dev.read(K).reshape(m, KV, D), dev.read(V).reshape(m, KV, D)
    see, mine = sees(np.arange(m), m, left, 0, sinks), slice(start[b], start[b] + m)
    check(run(dev, ic, q[mine], k, v, 0, left, 0, sinks, np.float32(D ** -0.5)), q[mine], k, v, see, np.float32(D ** -0.5))
    # Single tokens of all sequences, the layer recorded once.
    s, first = layer.held.seqs(np.arange(n + 1), lengths, table), np.arange(n + 1)
    dev.finish()
    dev.api.ocl_graph_begin(dev.pb)
    layer.launch(s, n)
    graph = dev.api.ocl_graph_end(dev.pb)
    try:
        for step in range(4):
            lengths = lengths + 1
            x = rng.standard_normal((n, C)).astype(np.float32)
            for buf, y in ((layer.X, x), (layer.P, lengths - 1), (s.bufs[1], lengths)):
                dev.write(buf, np.ascontiguousarray(y))
            dev.api.ocl_graph_launch(dev.pb, graph)
            layer.checked(x, first, lengths, table)
            dev.finish()
    finally:
        ic.lib().ocl_graph_free(graph)
