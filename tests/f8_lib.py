"""Weights in E4M3 with a scale for each block of 128 x 128 for the tests, x as
the products take it, and both in 64 bits."""

import numpy as np

BLOCK = 128


def table():
    """What each of E4M3's 256 bytes stands for."""
    byte = np.arange(256)
    e, m = (byte >> 3) & 15, byte & 7
    v = np.where(e == 0, m / 8.0 * 2.0 ** -6, (1 + m / 8.0) * 2.0 ** (e - 7.0))
    v = np.where((byte & 127) == 127, np.nan, v)
    return np.where(byte < 128, v, -v)


TABLE = table()


def random_weights(r, n, k, scale=0.03):
    """Bytes [n, k], any but NaN's, and scales [n / 128, k / 128] of both signs."""
    w = r.integers(0, 256, (n, k), dtype=np.uint8)
    w = np.where((w & 127) == 127, w ^ 1, w).astype(np.uint8)
    scales = r.uniform(0.1, 1.0, (-(-n // BLOCK), -(-k // BLOCK))) * scale / 448 * r.choice([-1.0, 1.0])
    return w, scales.astype(np.float32)


def widen(w, scales):
    """The weights [n, k] in float64."""
    n, k = w.shape
    s = scales.astype(np.float64).repeat(BLOCK, 0)[:n].repeat(BLOCK, 1)[:, :k]
    return TABLE[w] * s


def rounded(v):
    """Numbers of magnitude 448 at most to E4M3, ties to even."""
    a = np.abs(v)
    step = np.exp2(np.maximum(np.frexp(a)[1] - 1, -6) - 3.0)
    return np.rint(v / step) * step


def held(x):
    """x's numbers as a product takes them, in float64."""
    m, k = x.shape
    blocks = -(-k // BLOCK)
    g = np.zeros((m, blocks * BLOCK))
    g[:, :k] = x
    g = g.reshape(m, blocks, BLOCK)
    top = np.abs(g).max(-1, keepdims=True)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.maximum(np.ceil(np.log2(top / 448.0)), -101)
        e = np.where(top > 448 * np.exp2(e), e + 1, e)
        e = np.where((top <= 448 * np.exp2(e - 1)) & (e > -101), e - 1, e)
        q = rounded(g / np.exp2(e)) * np.exp2(e)
    q = np.where(np.isfinite(top), q, np.nan)
    return q.reshape(m, -1)[:, :k]


def exact(w, scales, x):
    """x' w^T and the sum of its products' magnitudes, in float64."""
    v, q = widen(w, scales), held(x)
    return q @ v.T, np.abs(q) @ np.abs(v).T


def bound(k, steps=0):
    """How far a product of k may lie from the exact one, of the sum of its
    products' magnitudes.  The products are exact in FP16 and the sum of a block's
    128 in single precision, each addition off by 2^-24 of what is summed so far at
    most, as the MFMA's order has them; then a block's scale times its power of two,
    a multiplication and an addition, up to 8 partial sums and the chain's steps."""
    return (128 + 3 * (-(-k // BLOCK)) + 8 + steps) * 2.0 ** -24
