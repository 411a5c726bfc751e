# SPDX-License-Identifier: Unlicense
"""GPU: the operators for long sequences as a transformer layer uses them:
query, key and value projections in 8 bits of one packed buffer, rotary
positions in place, the index, the selection and the attention over the
selected blocks, the output projection in 8 bits onto the residual; then a
token appended to the kept keys, values and index and computed alone.

Every step is held to its own definition on the inputs that it was given
(bounds of the operators' own tests), so that a rounding that moves a code or
a block in one of them is not an error of the next."""

import numpy as np
import pytest

import long_ref as ref
import test_q8_gpu as q8
from long_ref import U

pytestmark = pytest.mark.gpu


class Layer:
    def __init__(self, dev, ic, n, most, c=256, h=8, kv=4, d=32, bs=32, top=3):
        self.dev, self.ic, self.c, self.h, self.kv, self.d, self.bs, self.top = dev, ic, c, h, kv, d, bs, top
        rng = np.random.default_rng(n)
        self.wide = (h + 2 * kv) * d
        self.wqkv = (rng.standard_normal((self.wide, c)) * 1.5 / c ** 0.5).astype(np.float32)
        self.wo = (rng.standard_normal((c, h * d)) / (h * d) ** 0.5).astype(np.float32)
        self.freq = np.zeros(d // 2)
        ic.api().ops_rope_freqs(self.freq.ctypes.data, d, 2, 10000.0, 1, 2.0, 0.0, 0.0, 0.0)
        self.W = [self._weight(w) for w in (self.wqkv, self.wo)]
        self.F = dev.upload(self.freq)
        self.QKV = dev.zeros(most * self.wide)
        self.nblk = dev.api.ops_key_blocks(most, bs)
        self.KC, self.KS = dev.alloc(self.nblk * kv * ref.pitch(d)), dev.alloc(self.nblk * kv * 4)

    def _weight(self, w):
        W, Q, S = self.dev.upload(w), self.dev.alloc(len(w) * ref.pitch(w.shape[1])), self.dev.alloc(len(w) * 4)
        self.dev.api.ops_quant_rows(self.dev.po, *w.shape, W.mem, 0, w.shape[1], Q.mem, S.mem)
        return Q, S

    def run(self, x, pos, at, checked=True):
        """Tokens at rows at .. of the kept ones, one pass; every step checked."""
        dev, ic, a, n, h, kv, d = self.dev, self.ic, self.dev.api, len(x), self.h, self.kv, self.d
        w, nk, wide = h * d, at + len(x), self.wide
        X, P, O, Y = dev.upload(x), dev.upload(pos), dev.zeros(n * w), dev.upload(x)
        SEL = dev.alloc(n * h * self.top * 4)
        work = dev.alloc(max(a.ops_linear_q8_work_bytes(n, max(self.c, w)),
                             a.ops_block_select_work_bytes(n, h, self.nblk, self.top),
                             a.ops_attention_blocks_work_bytes(n, nk, h, kv, d, self.bs, self.top)))
        base = at * wide
        m = lambda o: ic.mat(self.QKV, base + o, wide)  # noqa: E731
        a.ops_linear_q8(dev.po, n, self.c, wide, X.mem, 0, self.c, self.W[0][0].mem, self.W[0][1].mem, None, None, 0,
                        self.QKV.mem, base, wide, 0, 0.0, work.mem)
        qkv = dev.read(self.QKV, n * wide, np.float32, 4 * base).reshape(n, wide)
        a.ops_rope_pos(dev.po, n, d, d, 2, P.mem, self.F.mem, 1.0, 1, m(0), m(0), h, m(w), m(w), kv)
        first = at // self.bs
        k0, v0 = ic.mat(self.QKV, w, wide), ic.mat(self.QKV, w + kv * d, wide)
        blocks = a.ops_key_blocks(nk, self.bs)
        a.ops_block_index(dev.po, k0, nk, kv, d, self.bs, None, first, blocks - first, self.KC.mem, self.KS.mem)
        a.ops_block_select(dev.po, m(0), n, h, kv, d, self.KC.mem, self.KS.mem, blocks, self.top, SEL.mem, work.mem)
        scale = float(np.float32(d ** -0.5))
        a.ops_attention_blocks(dev.po, m(0), k0, v0, ic.mat(O, 0, w), n, nk, h, kv, d, self.bs, self.top, SEL.mem,
                               scale, None, work.mem)
        a.ops_linear_q8(dev.po, n, w, self.c, O.mem, 0, w, self.W[1][0].mem, self.W[1][1].mem, None, Y.mem, 0, Y.mem,
                        0, self.c, 0, 0.0, work.mem)
        y = dev.read(Y, n * self.c).reshape(n, self.c)
        if not checked:
            return y
        want, bound = q8.expected(x, self.wqkv, None, None, 0, 0)
        assert np.all(np.abs(qkv - want) <= bound)
        every = dev.read(self.QKV, nk * wide).reshape(nk, wide)
        q, k, v = (every[:, o:o + g * d].reshape(nk, g, d) for o, g in ((0, h), (w, kv), (w + kv * d, kv)))
        turned = ref.rope(qkv[:, :w + kv * d].reshape(n, h + kv, d), pos, self.freq, d, True)
        got = np.concatenate([q[at:], k[at:]], 1)
        assert np.all(np.abs(got - turned) <= 12 * U * np.abs(qkv).max())
        assert np.array_equal(every[at:, w + kv * d:], qkv[:, w + kv * d:])
        kc, ks = ref.index(k, self.bs)
        assert np.array_equal(dev.read(self.KS, blocks * kv).reshape(blocks, kv), ks)
        sel = dev.read(SEL, n * h * self.top, np.int32).reshape(n, h, self.top)
        assert np.array_equal(sel, ref.select(q[at:], kc, ks, self.top))
        o = dev.read(O, n * w).reshape(n, h, d)
        want, bound = ref.attend(q[at:], k, v, sel, self.bs, scale)
        assert np.all(np.abs(o - want) <= bound + 1e-37)
        want, bound = q8.expected(o.reshape(n, w), self.wo, None, x, 0, 0)
        assert np.all(np.abs(y - want) <= bound)
        return y


@pytest.mark.parametrize("h,w", [(3, 5), (13, 11), (25, 24)])
def test_layer_and_appended_tokens(h, w, dev, ic):
    print(f"[long layer] {h} x {w}", flush=True)
    n = h * w
    rng = np.random.default_rng(n)
    x = rng.standard_normal((n + 2, 256)).astype(np.float32)
    pos = np.stack(np.divmod(np.arange(n + 2), w), 1).astype(np.int32)
    layer = Layer(dev, ic, n, n + 2)
    layer.run(x[:n], pos[:n], 0)
    for t in (n, n + 1):
        layer.run(x[t:t + 1], pos[t:t + 1], t)
