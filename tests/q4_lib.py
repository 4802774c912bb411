"""Weights in ggml's 4-bit blocks for the tests: random blocks of Q4_0 and
Q4_1, and the numbers they stand for in 64 bits."""

import numpy as np

BYTES = {"q4_0": 18, "q4_1": 20}


def random_blocks(r, kind, n, k, scale=0.03):
    """Bytes [n, k / 32, 18 or 20]: scales uniform in [-scale, scale] (Q4_0) or
    [0, scale] (Q4_1, whose least values are about -7.5 of them), nibbles uniform."""
    blocks = k // 32
    d = r.uniform(-scale if kind == "q4_0" else 0.0, scale, (n, blocks, 1)).astype(np.float16)
    heads = [d]
    if kind == "q4_1":
        heads.append((-7.5 * d + r.uniform(-scale, scale, d.shape)).astype(np.float16))
    nibbles = r.integers(0, 256, (n, blocks, 16), dtype=np.uint8)
    return np.concatenate([h.view(np.uint8).reshape(n, blocks, 2) for h in heads] + [nibbles], axis=2)


def widen(blocks):
    """The weights [n, k] and the magnitudes of the two parts a product adds
    up, |d (q - 8)| + |c| with w = d (q - 8) + c, in float64."""
    n, count, size = blocks.shape
    d = blocks[:, :, 0:2].copy().view(np.float16).astype(np.float64)
    nib = blocks[:, :, size - 16:]
    q = np.concatenate([nib & 15, nib >> 4], axis=2).astype(np.float64)
    if size == 18:
        w = d * (q - 8)
        parts = np.abs(w)
    else:
        m = blocks[:, :, 2:4].copy().view(np.float16).astype(np.float64)
        w = d * q + m
        parts = np.abs(d * (q - 8)) + np.abs(m + 8 * d)
    return w.reshape(n, -1), parts.reshape(n, -1)


def exact(blocks, x):
    """x w^T and the sum of its products' magnitudes, in float64."""
    w, parts = widen(blocks)
    x = x.astype(np.float64)
    return x @ w.T, np.abs(x) @ parts.T


def bound(k, steps=0):
    """How far a product of k may lie from the exact one, of the sum of its
    products' magnitudes: x in two FP16 parts is within 2^-22 of itself, or
    2^-25 of 2^-14 of its row's greatest where its low part is no normal
    number; a block's 64 products (both parts) are summed in single precision,
    each addition off by 2^-24 of what is summed so far at most, then k / 32
    blocks by two multiplications and two additions each (the scale and the
    offset), then up to 16 partial sums and the chain's steps."""
    return 2.0 ** -22 + (64 + 4 * (k // 32) + 16 + steps) * 2.0 ** -24
