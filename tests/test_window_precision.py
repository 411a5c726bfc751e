# SPDX-License-Identifier: Unlicense
"""CPU: the limit on what float32's errors come to together (kept_stats.limits)
rejects operands of fewer bits, at every shape that the GPU tests hold to it."""

import numpy as np
import pytest

import kept_stats
from kept_ref import sees
from test_window_edges_gpu import WIDE
from test_window_gpu import data


def bf16(x):
    bits = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((bits + 0x7fff + (bits >> 16 & 1)) & 0xffff0000).astype(np.uint32).view(np.float32)


PARTS = {"f16": lambda x: x.astype(np.float16).astype(np.float32), "bf16": bf16,
         "two of bf16": lambda x: bf16(x) + bf16(x - bf16(x))}


def test_rounding_to_bf16():
    x = np.array([1, 1 + 2 ** -8, 1 + 3 * 2 ** -8, 1 + 2 ** -8 + 2 ** -20, -3.14159, 0], np.float32)
    assert np.array_equal(bf16(x), np.array([1, 1, 1 + 2 ** -6, 1 + 2 ** -7, -3.140625, 0], np.float32))


@pytest.mark.parametrize("nq,nk,h,kv,d,left,right,sinks", WIDE)
def test_fewer_bits_are_seen(nq, nk, h, kv, d, left, right, sinks):
    q, k, v = data(nq, nk, h, kv, d)
    scale, rows = np.float32(d ** -0.5), np.arange(nq)[:: max(1, nq // 8)][:8]
    see = sees(rows + nk - nq, nk, left, right, sinks)
    q = q[rows]
    want, limit = kept_stats.attend(q, k, v, see, scale), kept_stats.limits(q, k, v, see, scale)
    for name, part in PARTS.items():
        rms, most = kept_stats.worst(kept_stats.attend(q, k, v, see, scale, part), want, limit)
        print(f"  {name}: {rms:.1f} of the limit, at most {most:.1f}")
        assert rms > 1, name
