"""The norms around a block with every choice of their operands -- a scale, a
bias, a gate, each there or not, scales from 0 or from 1 -- at widths that fill
their threads and that do not, against float64."""

import itertools

import numpy as np
import pytest
import torch

import sdhip
from helpers import dev, normal, rng, unwritten
from test_gpu_residual import U, norm64

KINDS = ["none", "layer", "rms"]
SCALES = 0.75, 1.5  # the branch's and the residual's
EPS = 1e-6


def bounds(v, kinds, ops, offset):
    """The sum and the norm after it in float64, and how far a right one may lie
    from each: 12 roundings of a number of the sum, 10 of the norm's, and what the
    sum's own carry through it."""
    y, r = (t.astype(np.float64) for t in v)
    w0, b0, gate, w1, b1 = (None if t is None else t.astype(np.float64) for t in ops)
    z, zs = norm64(kinds[0], y, EPS, w0, b0, offset)
    g = 1.0 if gate is None else gate
    s = SCALES[1] * r + SCALES[0] * g * z
    s_bound = 12 * U * (np.abs(SCALES[1] * r) + SCALES[0] * np.abs(g) * zs)
    n, ns = norm64(kinds[1], s, EPS, w1, b1, offset)
    through = s_bound
    if kinds[1] != "none":
        c = s - s.mean(-1, keepdims=True) if kinds[1] == "layer" else s
        scale = 1 / np.sqrt((c * c).mean(-1, keepdims=True) + EPS)
        rms = np.sqrt((s_bound * s_bound).mean(-1, keepdims=True))
        through = scale * (s_bound + rms + np.abs(c) * scale * rms)
    if w1 is not None:
        through = through * (np.abs(w1) + offset)
    return (s, s_bound), (n, 10 * U * ns + 1.01 * through)


@pytest.mark.gpu
@pytest.mark.parametrize("post", KINDS)
@pytest.mark.parametrize("pre", KINDS)
@pytest.mark.parametrize("dim", [28, 256, 491, 700, 1000, 1280, 1999, 4000, 5001, 8000, 16001, 17000])
def test_every_choice_of_operands(gpu, post, pre, dim):
    r = rng(dim)
    shape = (3, dim)
    v = normal(r, shape, 0.5), normal(r, shape, 0.3, 2.0)
    y, res = (dev(t, gpu) for t in v)
    every = [normal(r, (dim,), 1.0, 0.2), normal(r, (dim,), 0.0, 0.2), normal(r, (dim,), 0.5, 0.5),
             normal(r, (dim,), 1.0, 0.2), normal(r, (dim,), 0.0, 0.2)]
    on = [dev(t, gpu) for t in every]
    for there in itertools.product([False, True], repeat=5):
        w0, b0, gate, w1, b1 = (t if h else None for t, h in zip(on, there))
        ops = [t if h else None for t, h in zip(every, there)]
        for offset in (0.0, 1.0) if there[0] or there[3] else (0.0,):
            want = bounds(v, (post, pre), ops, offset)
            for keep in (True, False):
                s, o = unwritten(shape, gpu) if keep else None, unwritten(shape, gpu)
                sdhip.norm_residual(y, res, s, o, sdhip.row_norm(post, EPS, w0, b0, offset),
                                    sdhip.row_norm(pre, EPS, w1, b1, offset), gate, *SCALES)
                for got, (exact, allowed) in zip((s, o), want):
                    if got is not None:
                        err = np.abs(got.cpu().numpy() - exact)
                        assert np.isfinite(err).all() and (err <= allowed).all(), (there, offset, keep)
