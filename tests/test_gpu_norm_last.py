"""GROUP_NORM of channels-last tensors with its chain, on the device against
float64.  Bounds: a normed number is rounded four times (its differences from the
mean's two parts, the scale, their product), the chain's steps once each; SiLU's
slope is below 1.1 and its own error 8 roundings."""

import numpy as np
import pytest
import torch

import sdhip
from helpers import dev, rng, uniform


def reference(x, groups, eps):
    """x [n, h, w, c] in float64: ceil(c / groups) channels a group, the last ones' as many as are left."""
    x = x.astype(np.float64)
    per = -(-x.shape[-1] // groups)
    y = np.empty_like(x)
    for c in range(0, x.shape[-1], per):
        g = x[..., c:c + per]
        mean = g.mean(axis=(1, 2, 3), keepdims=True)
        d = g - mean
        y[..., c:c + per] = d / np.sqrt((d * d).mean(axis=(1, 2, 3), keepdims=True) + np.float64(np.float32(eps)))
    return y


def affine(v, scale, shift, silu):
    y = v * scale.astype(np.float64) + shift.astype(np.float64)
    err = 2.0 ** -24 * (6 * np.abs(v * scale) + 2 * np.abs(shift))
    if silu:
        y = y / (1.0 + np.exp(-y))
        err = 1.1 * err + 8 * 2.0 ** -24 * np.abs(y) + 2.0 ** -126
    return y, err


def view(shape, gpu, before, behind, pixel=0):
    """Images [n, h, w, c] with numbers around each pixel's channels that stay as they were."""
    n, h, w, c = shape
    buf = torch.full((n, h, w, before + c + behind), -7.25, device=gpu)
    return buf, buf[..., before:before + c]


def check(gpu, shape, groups, silu=False, eps=1e-5, x=None, xpad=(0, 0), ypad=(0, 0), seed=0, steps=True):
    n, h, w, c = shape
    r = rng(seed + c + h)
    x = uniform(r, shape, 2.0) + uniform(r, (c,), 1.0) if x is None else x
    x = x.astype(np.float32)
    scale, shift = uniform(r, (c,), 2.0), uniform(r, (c,), 1.0)
    _, xd = view(shape, gpu, *xpad)
    xd.copy_(torch.from_numpy(x))
    buf, yd = view(shape, gpu, *ypad)
    chain = [("mul", dev(scale, gpu)), ("add", dev(shift, gpu))] + ([("silu", None)] if silu else [])
    sdhip.group_norm_last(xd, yd, groups, eps, sdhip.epilogue(chain))
    torch.cuda.synchronize()
    y, err = affine(reference(x, groups, eps), scale, shift, silu)
    got = yd.cpu().numpy()
    worst = (np.abs(got - y) / err).max()
    print(f"{shape} {groups} groups, {xpad} {ypad}: {worst:.3g} of the bound", flush=True)
    assert (np.abs(got - y) <= err).all()
    yd.fill_(-7.25)
    assert (buf == -7.25).all()


SHAPES = [((1, 1, 1, 1), 1), ((1, 1, 1, 64), 32), ((2, 1, 1, 7), 3), ((2, 8, 8, 1280), 32), ((1, 5, 3, 320), 32), ((3, 7, 9, 30), 8),
          ((1, 64, 64, 320), 32), ((2, 33, 17, 96), 32), ((1, 100, 100, 32), 32), ((1, 3, 5, 2560), 32), ((2, 4, 4, 1300), 1),
          ((1, 9, 9, 5000), 2), ((5, 2, 2, 65), 65), ((1, 40, 30, 130), 32), ((2, 16, 16, 1920), 32), ((1, 200, 150, 128), 32),
          ((70, 2, 3, 16), 4), ((1, 1, 3000, 12), 3), ((1, 3000, 1, 10), 5), ((1, 20, 20, 33), 40)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", SHAPES)
@pytest.mark.parametrize("silu", [False, True])
def test_shapes(gpu, shape, groups, silu):
    check(gpu, shape, groups, silu)


@pytest.mark.gpu
@pytest.mark.parametrize("xpad,ypad", [((0, 3), (0, 0)), ((0, 0), (1, 2)), ((4, 4), (0, 8)), ((2, 2), (5, 0))])
@pytest.mark.parametrize("shape,groups", [((2, 8, 8, 64), 32), ((1, 40, 40, 96), 8), ((2, 5, 7, 30), 3)])
def test_channels_of_wider_tensors(gpu, shape, groups, xpad, ypad):
    check(gpu, shape, groups, True, xpad=xpad, ypad=ypad)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["offset", "great", "greatest", "small", "one number", "zero", "first far", "last far"])
@pytest.mark.parametrize("shape,groups", [((1, 4, 5, 64), 32), ((2, 60, 50, 64), 4), ((1, 30, 30, 30), 3)])
def test_values(gpu, kind, shape, groups):
    """Means far from 0, single precision's greatest and least numbers, groups of
    one number, a first (or last) number far from the others."""
    r = rng(11)
    x = uniform(r, shape, 1.0).astype(np.float64)
    eps = 1e-5
    if kind == "offset":
        x = x + 12345.0
    elif kind == "great":
        x = x * 1e20
    elif kind == "greatest":
        x = np.where(x > 0, 3.3e38, -3.3e38)
    elif kind == "small":
        x, eps = x * 2.0 ** -130, 0.0
    elif kind == "one number":
        x = np.full(shape, -0.7)
    elif kind == "zero":
        x = np.zeros(shape)
    elif kind == "first far":
        x[:, 0, 0] = 1e8
    else:
        x[:, -1, -1] = -1e8
    check(gpu, shape, groups, False, eps, x)


@pytest.mark.gpu
def test_infinities_and_nans_stay_in_their_groups(gpu):
    x = uniform(rng(1), (2, 30, 20, 64), 1.0)
    x[0, 3, 4, 5] = np.inf
    x[1, 0, 0, 63] = np.nan
    xd = dev(x, gpu)
    y = torch.empty_like(xd)
    sdhip.group_norm_last(xd, y, 16, 1e-5)
    bad = np.zeros(x.shape, bool)
    bad[0, ..., 4:8] = bad[1, ..., 60:] = True
    assert (np.isfinite(y.cpu().numpy()) == ~bad).all()


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", [((2, 8, 8, 64), 32), ((2, 50, 60, 96), 32), ((1, 9, 9, 30), 3)])
def test_chains(gpu, shape, groups):
    """Operands of every extent, up to six steps; tokens as images of one row."""
    n, h, w, c = shape
    r = rng(2)
    x = uniform(r, shape, 2.0)
    v = reference(x, groups, 1e-5)
    xd = dev(x, gpu)
    for extents in ((1, 1, 1, 1), (n, 1, 1, c), (1, h, 1, 1), (1, 1, w, c), (n, h, w, c), (n, 1, w, 1)):
        o = uniform(r, extents, 1.0)
        p = uniform(r, (c,), 1.0)
        steps = [("mul", dev(o, gpu)), ("add", dev(p, gpu)), ("add", dev(o, gpu)), ("mul", dev(p, gpu)), ("add", dev(o, gpu))]
        y = torch.full(shape, float("nan"), device=gpu)
        sdhip.group_norm_last(xd, y, groups, 1e-5, sdhip.epilogue(steps))
        torch.cuda.synchronize()
        o64, p64 = o.astype(np.float64), p.astype(np.float64)
        want = (v * o64 + p64 + o64) * p64 + o64
        assert (np.abs(y.cpu().numpy() - want) <= 2.0 ** -24 * 10 * (np.abs(v) + 3)).all()
    tokens = torch.empty((n, h * w, c), device=gpu)
    image = torch.empty_like(xd)
    sdhip.group_norm_last(xd.view(n, h * w, c), tokens, groups, 1e-5)
    sdhip.group_norm_last(xd, image, groups, 1e-5)
    assert torch.equal(tokens.view(shape), image)
    sdhip.set_tuning("fuse=0")
    try:
        apart, fused = torch.empty_like(xd), torch.empty_like(xd)
        chain = sdhip.epilogue([("mul", dev(p, gpu)), ("silu", None)])
        sdhip.group_norm_last(xd, apart, groups, 1e-5, chain)
        sdhip.set_tuning("")
        sdhip.group_norm_last(xd, fused, groups, 1e-5, chain)
        # Each SiLU is within 8 roundings.
        assert ((apart - fused).abs() <= 16 * 2.0 ** -24 * fused.abs() + 2.0 ** -126).all()
    finally:
        sdhip.set_tuning("")


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", SHAPES)
def test_in_place_and_again(gpu, shape, groups):
    """In x's own memory, and the same bits every time."""
    x = dev(uniform(rng(3), shape, 2.0), gpu)
    y, z = torch.empty_like(x), torch.empty_like(x)
    sdhip.group_norm_last(x, y, groups, 1e-5)
    sdhip.group_norm_last(x, z, groups, 1e-5)
    sdhip.group_norm_last(x, x, groups, 1e-5)
    assert torch.equal(y, z) and torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", [((2, 8, 8, 64), 32), ((1, 90, 60, 96), 32)])
def test_captured_and_replayed(gpu, shape, groups):
    x, y, eager = (torch.zeros(shape, device=gpu) for _ in range(3))
    work = sdhip.group_norm_last(x, y, groups, 1e-5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sdhip.group_norm_last(x, y, groups, 1e-5, work=work)
    for i in range(3):
        x.copy_(dev(uniform(rng(i), shape, 1.0), gpu))
        sdhip.group_norm_last(x, eager, groups, 1e-5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager)


@pytest.mark.gpu
def test_many_images(gpu):
    """More images than one launch's workgroups are counted for here, each as alone."""
    x = dev(uniform(rng(4), (30000, 1, 2, 8), 1.0), gpu)
    y, one = torch.empty_like(x), torch.empty_like(x[:1])
    sdhip.group_norm_last(x, y, 2, 1e-5)
    for i in (0, 1, 29999):
        sdhip.group_norm_last(x[i:i + 1], one, 2, 1e-5)
        assert torch.allclose(one, y[i:i + 1], rtol=0, atol=2.0 ** -22)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", [((3, 1, 100003, 64), 32), ((3, 69, 565, 96), 32), ((1, 1, 263001, 12), 3), ((2, 1, 70001, 30), 3)])
def test_pixels_that_no_even_chunks_hold(gpu, shape, groups):
    """Chunks of as many pixels as the most wanted would leave the last of them none."""
    check(gpu, shape, groups)
