# SPDX-License-Identifier: Unlicense
"""CPU: offsets, and row counts and strides, whose bytes do not fit in 64 bits
are refused like any other access past a buffer. The addresses are never
dereferenced."""

import pytest
from test_long_refusals import env, refused  # noqa: F401  (env is a fixture)

# Rows times stride: some 2^62 floats (2^64 bytes), 2^61 (2^63) and just under.
FAR = [(2 ** 31 - 1, 2 ** 31 - 1), (2 ** 30 + 1, 2 ** 31 - 1), (2 ** 30 + 2, 2 ** 31 - 1), (2 ** 30, 2 ** 31 - 1)]


@pytest.mark.parametrize("rows,ld", FAR)
def test_rows_of_a_norm(rows, ld, ic, env):  # noqa: F811
    a, o, v = env
    G = 1 << 34
    none, far, near = ic.Opnd(None, 0, 0, 0, 0), ic.Opnd(v(0, G), 0, ld, 0, 0), ic.Opnd(v(G, G), 0, 1, 0, 0)
    q, s = v(2 * G, 64 * rows), v(64 * G, 4 * rows)
    for x, r, h, y, name in ((far, none, none, none, "X"), (near, far, none, none, "R"), (near, none, far, none, "H"),
                             (near, none, none, far, "Y")):
        with refused(ic, f"ops_rms_norm: {name} accessed"):
            a.ops_rms_norm(o, rows, 1, x, r, None, 1e-6, h, y, q, s)


@pytest.mark.parametrize("rows,ld", FAR)
def test_rows_of_codes(rows, ld, ic, env):  # noqa: F811
    a, o, v = env
    with refused(ic, "ops_quant_rows: X accessed"):
        a.ops_quant_rows(o, rows, 1, v(0, 1 << 20), 0, ld, v(1 << 34, 64 * rows), v(1 << 40, 4 * rows))


@pytest.mark.parametrize("off", [2 ** 61, 2 ** 62, 2 ** 62 + 8, 2 ** 63 - 1])
def test_offsets(off, ic, env):  # noqa: F811
    """2^62 floats on is the buffer's start again in 64 bits, 2^63 - 1 four bytes
    before it."""
    a, o, v = env
    none, y = ic.Opnd(None, 0, 0, 0, 0), ic.Opnd(v(1 << 30, 4000), 0, 100, 0, 0)
    with refused(ic, "ops_rms_norm: X accessed"):
        a.ops_rms_norm(o, 10, 100, ic.Opnd(v(0, 4000), off, 100, 0, 0), none, None, 1e-6, none, y, None, None)
