# SPDX-License-Identifier: Unlicense
"""What rounding errors of attention come to together, beside the worst case of
kept_ref.attend: on normally distributed operands they have no common sign, and
lost bits of the operands show long before they pass the worst case."""

import numpy as np

from long_ref import U


def weights(q, k, see, scale):
    """Per head (queries, keys): scores to base 2, softmax weights, and the root
    of the sum of a score's squared products; 64 bits."""
    g = q.shape[1] // k.shape[1]
    for i in range(q.shape[1]):
        a, b = q[:, i].astype(np.float64) * (float(scale) * np.log2(np.e)), k[:, i // g].astype(np.float64)
        s = np.where(see, a @ b.T, -np.inf)
        p = np.exp2(s - s.max(1, keepdims=True))
        yield s, p / p.sum(1, keepdims=True), np.sqrt((a * a) @ (b * b).T)


def attend(q, k, v, see, scale, part=lambda x: x):
    """The attention in 64 bits, each operand rounded once by `part`."""
    g, out = q.shape[1] // k.shape[1], np.zeros(q.shape)
    for i, (_, p, _) in enumerate(weights(part(q * np.float32(1)), part(k), see, scale)):
        out[:, i] = part(p.astype(np.float32)).astype(np.float64) @ part(v[:, i // g]).astype(np.float64)
    return out


def limits(q, k, v, see, scale):
    """(queries, heads): root mean square over a row's channels that float32's
    errors come to, from what each adds in quadrature. An output is sum p v; an
    error e of a score changes it by p e (v - o), so that of independent ones sqrt(sum p^2
    e^2) times the values' deviation stays, which over sqrt(sum p^2) is e's root
    mean square with weights p^2. A score's sum is rounded d times by up to U of
    itself (less on the way there, as many have one sign as the other: sqrt(d) / 2
    of U |s|), and its operands to 22 bits, 4 U of each product (4 U of the products'
    root sum of squares). The weights and their products with values, to 22
    bits, and exponentials add 8 U, the sums over n keys sqrt(n) / 2 of U."""
    out = np.zeros(q.shape[:2])
    n = see.sum(1)
    for i, (s, p, size) in enumerate(weights(q, k, see, scale)):
        p2 = p * p
        mean = lambda x: np.sqrt((p2 * np.where(see, x, 0) ** 2).sum(1) / p2.sum(1))  # noqa: E731
        dev = np.sqrt(p2.sum(1)) * np.abs(v).std()
        out[:, i] = U * (np.sqrt(q.shape[2]) / 2 * mean(np.where(see, s, 0)) + 4 * mean(size) + np.sqrt(n) / 2 + 8) * dev
    return out


def worst(got, want, limit):
    """(a case's root mean square, its largest error) over the limit: at most 1
    and, of so many values of rows unlike one another, 12."""
    err = (got - want) / limit[..., None]
    return np.sqrt((err ** 2).mean()), np.abs(err).max()
