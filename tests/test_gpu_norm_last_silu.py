"""SiLU after the channels-last norm over its whole range, on the device, by one
launch, two and three, against float64 and against the chain apart (fuse = 0).

Bounds: SiLU's own error is 7 roundings of 2^-24, 8 with its square, and from
-87.33 on, where 1 + exp(-x) passes 2^126, |x| 2^-126 (the chain apart, whose power
stops at exp(88.73), as much); that of its argument goes through its slope, below
1.1.  Of zeros the norm is 0, so that the argument is the shift as it is."""

import numpy as np
import pytest
import torch

import sdhip
from helpers import dev, rng, uniform
from test_gpu_norm_last import reference

# Images [n, h, w, c], groups, and what their calls take.
FORMS = {"one launch": ((1, 2, 2, 128), 32), "two launches": ((2, 60, 50, 128), 32), "three launches": ((1, 200, 150, 128), 32),
         "single channels": ((1, 20, 20, 129), 3), "wide channels, two launches": ((1, 40, 50, 130), 32)}


def silu_of(v):
    with np.errstate(over="ignore"):
        return v / (1.0 + np.exp(-v))


def tail(v):
    return 2.0 ** -126 * np.where(v < -87.3, np.abs(v), 1.0)


def call(xd, groups, steps, apart=False):
    y = torch.full(xd.shape, float("nan"), device=xd.device)
    if apart:
        sdhip.set_tuning("fuse=0")
    try:
        sdhip.group_norm_last(xd, y, groups, 1e-5, sdhip.epilogue(steps))
    finally:
        sdhip.set_tuning("")
    torch.cuda.synchronize()
    return y.cpu().numpy()


def arguments():
    """Numbers along SiLU's range, most of them around where its power overflows."""
    edge = np.arange(*(np.float32(v).view(np.uint32) for v in (-88.71, -88.74)), dtype=np.uint32).view(np.float32)
    parts = [np.linspace(-1e5, 1e5, 2048), np.linspace(-130, -80, 4096), np.linspace(-2000, 2000, 2048), np.linspace(-20, 20, 4096),
             np.linspace(-3.4e38, 3.4e38, 512), edge, [0.0, -0.0, 1e-40, -1e-40, 88.72, 88.73, 126.0, 2.5e38]]
    return np.concatenate([np.asarray(p, np.float32) for p in parts])


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS)
def test_work_buffers(gpu, form):
    """The shapes take the launches they are named for: none of one, sums of the parts, and the joined too."""
    (n, h, w, c), groups = FORMS[form]
    x = torch.empty((n, h, w, c), device=gpu)
    real = -(-c // -(-c // groups))
    doubles = sdhip.load().sdhip_group_norm_last_work_size(sdhip.desc(x), sdhip.desc(x), groups) // (8 * n * real)
    if "launches" not in form:
        assert doubles == 0
    elif form.startswith("three"):
        assert doubles > 2 * 256 + 1
    else:
        assert 0 < doubles <= 2 * 256 + 1


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS)
def test_every_argument(gpu, form):
    shape, groups = FORMS[form]
    c = shape[-1]
    all_of = arguments()
    values = np.resize(all_of, -(-all_of.size // c) * c).reshape(-1, c)
    xd = torch.zeros(shape, device=gpu)
    worst = 0.0
    for i in range(0, len(values), 1 if form == "one launch" else 8):  # every 8th row of them by the larger images
        v = values[i].astype(np.float64)
        want, err = silu_of(v), 8 * 2.0 ** -24 * np.abs(silu_of(v)) + tail(v)
        steps = [("add", dev(values[i], gpu)), ("silu", None)]
        y = call(xd, groups, steps)
        off = np.abs(y - want)
        assert (off <= err).all(), (values[i][~(off <= err).all(axis=(0, 1, 2))], y[0, 0, 0][~(off <= err).all(axis=(0, 1, 2))])
        worst = max(worst, (off / np.where(v < -87.3, np.inf, 2.0 ** -24 * np.abs(want) + 2.0 ** -126)).max())
        apart = call(xd, groups, steps, apart=True)
        assert (np.abs(apart.astype(np.float64) - y) <= 2 * err).all()
    print(f"{form}: {worst:.2f} roundings", flush=True)


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS)
def test_outliers_and_great_scales(gpu, form):
    """What reaches there in earnest: a group of one far number, scaled to 1e5 and more."""
    shape, groups = FORMS[form]
    c = shape[-1]
    r = rng(21)
    x = uniform(r, shape, 1.0)
    x[0, 0, 0, ::3] = 1e4
    x[-1, -1, -1, 1::3] = -1e4
    normed = reference(x, groups, 1e-5)
    for most in (1.0, 30.0, 3000.0, 1e5):
        scale = (uniform(r, (c,), 1.0) * most).astype(np.float32)
        shift = uniform(r, (c,), 100.0).astype(np.float32)
        v = normed * scale + shift
        want = silu_of(v)
        err = (1.1 * 2.0 ** -24 * (6 * np.abs(normed * scale) + 2 * np.abs(shift)) + 8 * 2.0 ** -24 * np.abs(want)
               + 2.0 ** -126 * np.maximum(np.abs(v), 1.0))
        xd, steps = dev(x, gpu), [("mul", dev(scale, gpu)), ("add", dev(shift, gpu)), ("silu", None)]
        y = call(xd, groups, steps)
        assert (np.abs(y - want) <= err).all()
        assert (np.abs(call(xd, groups, steps, apart=True) - y) <= 2 * err).all()


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS)
def test_infinite_and_nan_shifts(gpu, form):
    shape, groups = FORMS[form]
    shift = np.zeros(shape[-1], np.float32)
    shift[1], shift[2] = np.inf, np.nan
    xd = torch.zeros(shape, device=gpu)
    for apart in (False, True):
        y = call(xd, groups, [("add", dev(shift, gpu)), ("silu", None)], apart)
        assert (y[..., 1] == np.inf).all() and np.isnan(y[..., 2]).all()
        assert (y[..., 0] == 0).all() and (y[..., 3:] == 0).all()
