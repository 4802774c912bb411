"""Rotary positions of several axes after the heads' norm, on the device against
float64.  Bounds: a sine or cosine is within 4 x 2^-24 (its argument's rounding and
its own), a turned number two products and an addition of such, a normed one
8 roundings before that (its difference from the mean in two parts, the root, the
weight and its offset, the products, the bias); FP16 outputs half a step more."""

import numpy as np
import pytest
import torch

import sdhip
from helpers import dev, rng, uniform


def reference(x, at, dims, base, order, shared=False, norm=None, eps=1e-6, weight=None, bias=None, offset=0.0):
    """x [b, h, l, d], at [b or 1, l or 1, axes]: y, and the magnitudes that its errors are of."""
    z = x.astype(np.float64)
    if norm == "layer":
        z = z - z.mean(-1, keepdims=True)
    if norm is not None:
        z = z / np.sqrt((z * z).mean(-1, keepdims=True) + eps)
    z = z * (weight + offset) if weight is not None else z
    mag = np.abs(z) + (np.abs(bias) if bias is not None else 0.0)
    z = z + bias if bias is not None else z
    y, size = z.copy(), mag.copy()
    n, p = sum(dims), 0
    bases = [base] * len(dims) if np.isscalar(base) else base
    for a, d in enumerate(dims):
        for j in range(d // 2):
            f = float(np.float32(bases[a])) ** (-2.0 * p / n if shared else -2.0 * j / d)
            t = at[:, None, :, a].astype(np.float64) * f
            i, k = (2 * p, 2 * p + 1) if order == "adjacent" else (p, n // 2 + p)
            y[..., i], y[..., k] = z[..., i] * np.cos(t) - z[..., k] * np.sin(t), z[..., i] * np.sin(t) + z[..., k] * np.cos(t)
            size[..., i] = size[..., k] = mag[..., i] + mag[..., k]
            p += 1
    return y, size


def allowed(y, size, half):
    return 16 * 2.0 ** -24 * size + (2.0 ** -11 * np.abs(y) + 2.0 ** -25 if half else 0.0) * 1.001


def laid(shape, kind, device, dtype=torch.float32):
    """A tensor [b, h, l, d] laid out as a caller may hold it, in numbers that stay as they were."""
    b, h, l, d = shape
    if kind == "heads":        # [b, h, l, d] as it is
        buf = torch.full((b * h * l * d + 64,), -7.25, device=device, dtype=dtype)
        t = buf[32:32 + b * h * l * d].view(b, h, l, d)
    elif kind == "tokens":     # [b, l, h, d]
        buf = torch.full((b * h * l * d + 64,), -7.25, device=device, dtype=dtype)
        t = buf[32:32 + b * h * l * d].view(b, l, h, d).permute(0, 2, 1, 3)
    elif kind == "projection":  # heads among others' in a projection's output
        buf = torch.full((b, l, 2 * h * d + 8), -7.25, device=device, dtype=dtype)
        t = torch.as_strided(buf, (b, h, l, d), (buf.stride(0), d, buf.stride(1), 1), 4)
    else:                      # "odd": rows at odd multiples of their size
        buf = torch.full((b, l, h, d + 1), -7.25, device=device, dtype=dtype)
        t = buf[..., 1:].permute(0, 2, 1, 3)
    return buf, t


def check(gpu, shape, dims, base=10000.0, order="adjacent", shared=False, norm=None, layout=("tokens", "tokens"), half=False,
          at=None, weight=None, bias=None, offset=0.0, x=None, eps=1e-6, seed=1):
    b, h, l, d = shape
    r = rng(seed + l + d)
    x = uniform(r, shape, 2.0) if x is None else x
    at = np.floor(r.uniform(0, 100, (1, l, len(dims)))).astype(np.float32) if at is None else at
    _, xd = laid(shape, layout[0], gpu)
    xd.copy_(torch.from_numpy(x))
    buf, yd = laid(shape, layout[1], gpu, torch.float16 if half else torch.float32)
    before = buf.clone()
    # The operands as they are given, and spread over [b, h, l, d].
    spread = {n: None if v is None else v.astype(np.float64) for n, v in (("weight", weight), ("bias", bias))}
    n = None
    if norm is not None or weight is not None or bias is not None:
        n = sdhip.row_norm(norm or "none", eps, None if weight is None else dev(weight, gpu), None if bias is None else dev(bias, gpu), offset)
    sdhip.rope(xd, dev(at, gpu), sdhip.rope_axes(dims, base, order, shared), yd, n)
    torch.cuda.synchronize()
    y, size = reference(x, at, dims, base, order, shared, norm, np.float64(np.float32(eps)), offset=offset, **spread)
    got = yd.cpu().numpy().astype(np.float64)
    with np.errstate(invalid="ignore"):  # 0 of 0
        worst = np.nan_to_num(np.abs(got - y) / allowed(y, size, half)).max()
    print(f"{shape} {dims} {order} {norm} {layout} half {half}: {worst:.3g} of the bound", flush=True)
    assert (np.abs(got - y) <= allowed(y, size, half)).all()
    assert xd.cpu().numpy().tobytes() == x.tobytes() or np.array_equal(xd.cpu().numpy(), x, equal_nan=True)
    yd.fill_(0.0)
    torch.as_strided(before, yd.shape, yd.stride(), yd.storage_offset()).fill_(0.0)
    assert torch.equal(buf, before)  # nothing but y is written


ORDERS = ["adjacent", "halves"]
LAYOUTS = [("tokens", "tokens"), ("projection", "heads"), ("heads", "projection"), ("odd", "tokens"), ("tokens", "odd"), ("odd", "odd")]


@pytest.mark.gpu
@pytest.mark.parametrize("order", ORDERS)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("d,dims", [(2, [2]), (3, [2]), (8, [8]), (40, [40]), (64, [32, 32]), (72, [24, 24, 24]), (80, [80]),
                                    (96, [10, 22, 40]), (128, [16, 56, 56]), (128, [44, 42, 42]), (130, [2, 4, 6, 8]), (160, [96, 64]),
                                    (256, [128]), (300, [298, 2]), (500, [500]), (511, [510]), (512, [508]), (512, [128, 128, 128, 128])])
def test_heads_and_axes(gpu, order, layout, d, dims):
    check(gpu, (2, 3, 5, d), dims, order=order, layout=layout, seed=d)
    check(gpu, (1, 5, 3, d), dims, order=order, layout=layout, seed=d, norm="rms", half=True)


@pytest.mark.gpu
@pytest.mark.parametrize("order", ORDERS)
@pytest.mark.parametrize("shape", [(1, 1, 1, 128), (1, 32, 1, 128), (1, 1, 1000, 64), (3, 7, 77, 64), (2, 24, 300, 128), (1, 200, 2, 96)])
@pytest.mark.parametrize("norm", [None, "rms", "layer"])
def test_tokens_and_heads(gpu, order, shape, norm):
    d = shape[3]
    r = rng(d)
    weight = uniform(r, (shape[1], 1, d), 1.0) if norm else None
    bias = uniform(r, (d,), 1.0) if norm == "layer" else None
    check(gpu, shape, [d // 4, d // 4, d // 2], order=order, norm=norm, weight=weight, bias=bias, layout=("projection", "tokens"))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [None, "rms", "layer"])
@pytest.mark.parametrize("extents", [(1, 1, 1, 96), (1, 1, 1, 1), (2, 1, 1, 96), (1, 3, 1, 1), (1, 1, 7, 96), (2, 3, 7, 96)])
def test_operands_of_every_extent(gpu, kind, extents):
    r = rng(sum(extents))
    check(gpu, (2, 3, 7, 96), [32, 32], norm=kind, weight=uniform(r, extents, 1.0), bias=uniform(r, extents, 1.0), offset=1.0)
    check(gpu, (2, 3, 7, 95), [32, 30], norm=kind, weight=uniform(r, extents[:3] + (min(95, extents[3]),), 1.0), order="halves")


@pytest.mark.gpu
@pytest.mark.parametrize("order", ORDERS)
@pytest.mark.parametrize("shared", [False, True])
def test_positions(gpu, order, shared):
    """Far, fractional and negative positions, a base for each axis, positions of
    each batch or of all tokens alike."""
    r = rng(3)
    shape, dims = (3, 2, 9, 64), [16, 24, 24]
    for at in (uniform(r, (1, 9, 3), 2.0 ** 24), np.rint(uniform(r, (3, 9, 3), 1e6)), uniform(r, (3, 9, 3), 0.5),
               uniform(r, (3, 1, 3), 50.0), uniform(r, (1, 1, 3), 1e9), np.zeros((1, 9, 3))):
        check(gpu, shape, dims, base=[100.0, 10000.0, 1e6], order=order, shared=shared, at=at.astype(np.float32))
    check(gpu, shape, dims, base=0.5, order=order, shared=shared)
    check(gpu, shape, dims, base=1.0, order=order, shared=shared)


@pytest.mark.gpu
def test_positions_of_zero_change_nothing(gpu):
    x = dev(uniform(rng(1), (1, 4, 6, 128), 1.0), gpu)
    y = torch.empty_like(x)
    sdhip.rope(x, torch.zeros((6, 2), device=gpu), sdhip.rope_axes([64, 64]), y)
    assert torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("order", ORDERS)
def test_infinities_stay_with_their_pairs(gpu, order):
    """Numbers that are not turned, and pairs, keep to themselves."""
    d, n = 80, 64
    x = uniform(rng(2), (1, 2, 3, d), 1.0)
    x[0, 0, 1, 70] = np.inf
    x[0, 1, 2, 79] = np.nan
    x[0, 0, 2, 5] = np.inf
    xd, at = dev(x, gpu), dev(uniform(rng(4), (3, 2), 9.0), gpu)
    y = torch.empty_like(xd)
    sdhip.rope(xd, at, sdhip.rope_axes([32, 32], order=order), y)
    got = y.cpu().numpy()
    want = np.zeros(x.shape, bool)
    want[0, 0, 1, 70] = want[0, 1, 2, 79] = True
    want[0, 0, 2, [4, 5] if order == "adjacent" else [5, 5 + n // 2]] = True
    assert (np.isfinite(got) == ~want).all()
    assert got[0, 0, 1, 70] == np.inf and np.isnan(got[0, 1, 2, 79])
    # A position that is no number turns its own token's pairs to NaN.
    at[1, 0] = float("nan")
    sdhip.rope(dev(uniform(rng(2), x.shape, 1.0), gpu), at, sdhip.rope_axes([32, 32], order=order), y)
    nan = np.isnan(y.cpu().numpy())
    assert nan[:, :, 1].sum() == 2 * 32 and not nan[:, :, [0, 2]].any() and not nan[..., n:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("power", [-140, -60, 0, 60, 126])
def test_rows_of_any_magnitude(gpu, norm, power):
    x = (uniform(rng(5), (1, 3, 4, 64), 1.0).astype(np.float64) * 2.0 ** power).astype(np.float32)
    check(gpu, x.shape, [64], norm=norm, x=x, eps=0.0)
    flat = np.full((1, 3, 4, 64), 3.0 * 2.0 ** power, np.float32)
    check(gpu, flat.shape, [64], norm=norm, x=flat, eps=1e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("order", ORDERS)
@pytest.mark.parametrize("d", [33, 64, 128, 512])
def test_in_place(gpu, order, d):
    x = dev(uniform(rng(6), (2, 4, 5, d), 1.0), gpu)
    at, axes = dev(uniform(rng(7), (5, 2), 30.0), gpu), sdhip.rope_axes([16, 8], order=order)
    n = sdhip.row_norm("rms", 1e-6, dev(uniform(rng(8), (d,), 1.0), gpu))
    y = torch.empty_like(x)
    sdhip.rope(x, at, axes, y, n)
    sdhip.rope(x, at, axes, x, n)
    assert torch.equal(x, y)


@pytest.mark.gpu
def test_captured_and_replayed(gpu):
    shape = (1, 6, 50, 64)
    x, at, y, eager = (torch.zeros(s, device=gpu) for s in (shape, (50, 2), shape, shape))
    axes = sdhip.rope_axes([32, 32])
    sdhip.rope(x, at, axes, y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sdhip.rope(x, at, axes, y)
    for i in range(3):
        x.copy_(dev(uniform(rng(i), shape, 1.0), gpu))
        at.copy_(dev(uniform(rng(i), (50, 2), 1000.0), gpu))
        sdhip.rope(x, at, axes, eager)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager)


@pytest.mark.gpu
def test_many_tokens(gpu):
    """More tokens than the device has waves, each as it is alone."""
    x = dev(uniform(rng(9), (2, 2, 40000, 32), 1.0), gpu)
    at = torch.arange(40000, device=gpu, dtype=torch.float32)[:, None]
    y, one = torch.empty_like(x), torch.empty((2, 2, 1, 32), device=gpu)
    sdhip.rope(x, at, sdhip.rope_axes([32]), y)
    for l in (0, 1, 4097, 39999):
        sdhip.rope(x[:, :, l:l + 1], at[l:l + 1], sdhip.rope_axes([32]), one)
        assert torch.equal(one, y[:, :, l:l + 1])


@pytest.mark.gpu
@pytest.mark.parametrize("order", ORDERS)
@pytest.mark.parametrize("norm", [None, "rms", "layer"])
@pytest.mark.parametrize("shape,dims", [((1, 1, 5000, 64), [64]), ((2500, 1, 2, 40), [16, 8]), ((3, 2, 1501, 128), [40, 42, 46]), ((2, 4, 2100, 64), [2, 62]),
                                        ((7, 3, 601, 33), [30]), ((4999, 1, 1, 72), [72])])
def test_many_tokens_of_few_heads(gpu, order, norm, shape, dims):
    """Rows of several tokens, and batches, by a wave; weights and offsets a head, strides of any kind."""
    b, h, l, d = shape
    r = rng(l)
    weight, bias = uniform(r, (1, h, 1, d), 2.0), uniform(r, (b, 1, 1, d), 1.0)
    for layout in (("tokens", "tokens"), ("projection", "odd")):
        check(gpu, shape, dims, order=order, norm=norm, weight=weight, bias=bias, layout=layout, half=layout[1] == "tokens",
              at=np.floor(r.uniform(0, 100, (b, l, len(dims)))).astype(np.float32))
