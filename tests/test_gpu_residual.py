"""The norms after and before a block with its gate and residual
(sdhip_norm_residual) on the device against float64."""

import numpy as np
import pytest
import torch

import sdhip
from helpers import dev, normal, rng, unwritten

U = 2.0 ** -24  # half a step of single precision


def norm64(kind, v, eps, weight, bias, offset):
    """The norm, and the magnitudes its roundings are of."""
    size = np.abs(v)
    if kind == "layer":
        mean = v.mean(-1, keepdims=True)
        v = v - mean
        size = np.abs(v) + 2.0 ** -20 * np.abs(mean)  # the mean's second part is held to 2^-48 of it
    if kind != "none":
        scale = 1 / np.sqrt((v * v).mean(-1, keepdims=True) + eps)
        v, size = v * scale, size * scale
    if weight is not None:
        v, size = v * (weight + offset), size * (np.abs(weight) + abs(offset))
    if bias is not None:
        v, size = v + bias, size + np.abs(bias)
    return v, size


def run(gpu, shape, post="rms", pre="rms", modulated=False, bias=True, gate=True, sum=True, out=True, y=True, seed=1,
        eps=1e-6, scales=(0.75, 1.5), y_np=None, r_np=None, place=None):
    """One call; the numbers it wrote and what they should be, with bounds."""
    r = rng(seed)
    dim = shape[-1]
    y_np = normal(r, shape) if y_np is None else y_np
    r_np = normal(r, shape, 0.3, 2.0) if r_np is None else r_np
    wide = (shape[0],) + (1,) * (len(shape) - 2) + (dim,) if modulated else (dim,)
    offset = 1.0 if modulated else 0.0
    ops = {n: normal(r, wide, 0.0 if modulated else 1.0, 0.2) for n in ("w0", "w1")}
    ops.update({n: normal(r, wide, 0.0, 0.2) for n in ("b0", "b1")} if bias else {})
    if gate:
        ops["gate"] = normal(r, wide, 0.0, 0.5)
    d = {n: dev(v, gpu) for n, v in ops.items()}
    yd, rd = dev(y_np, gpu), dev(r_np, gpu)
    sd = unwritten(shape, gpu) if sum else None
    od = unwritten(shape, gpu) if out else None
    if place is not None:
        yd, rd, sd, od = place(yd, rd, sd, od)
    post_n = sdhip.row_norm(post, eps, d["w0"], d.get("b0"), offset) if y else None
    pre_n = sdhip.row_norm(pre, eps, d["w1"], d.get("b1"), offset) if out else None
    sdhip.norm_residual(yd if y else None, rd, sd, od, post_n, pre_n, d.get("gate") if y else None, *scales)
    torch.cuda.synchronize()
    f = {n: v.astype(np.float64) for n, v in ops.items()}
    s = r_np.astype(np.float64) * scales[1]
    size = np.abs(s)
    if y:
        z, zs = norm64(post, y_np.astype(np.float64), eps, f["w0"], f.get("b0"), offset)
        g = f["gate"] if gate else 1.0
        s, size = s + scales[0] * g * z, size + abs(scales[0]) * np.abs(g) * zs
    # A number of s takes 10 roundings at most: of v - mean (2), the scale (2), their product, weight + offset, its
    # product, the bias, the gate, the scale and the sum.
    s_bound = 12 * U * size
    results = {}
    if sum:
        results["sum"] = (sd.cpu().numpy(), s, s_bound)
    if out:
        n, ns = norm64(pre, s, eps, f["w1"], f.get("b1"), offset)
        # s's own error passes through the norm: times its scale at each number, and by the mean and the scale, which
        # move no further than the root of the errors' mean square does.
        if pre == "none":
            through = s_bound
        else:
            c = s - s.mean(-1, keepdims=True) if pre == "layer" else s
            scale = 1 / np.sqrt((c * c).mean(-1, keepdims=True) + eps)
            rms = np.sqrt((s_bound * s_bound).mean(-1, keepdims=True))
            through = scale * (s_bound + rms + np.abs(c) * scale * rms)
        through = through * (np.abs(f["w1"]) + offset)
        results["out"] = (od.cpu().numpy(), n, 10 * U * ns + 1.01 * through)
    return results


def check(results, what):
    for name, (got, want, allowed) in results.items():
        assert np.isfinite(got).all(), (what, name)
        worst = (np.abs(got - want) / (allowed + 1e-37)).max()
        print(f"{what} {name}: {worst:.3g} of the bound")
        assert worst <= 1.0, (what, name)


KINDS = ["none", "layer", "rms"]
DIMS = [1, 2, 3, 4, 31, 63, 64, 65, 127, 128, 252, 256, 257, 320, 513, 768, 1021, 1024, 1280, 1532, 2048, 2049, 4096, 5120,
        5121, 8192, 10240, 16384, 16385, 20000]


@pytest.mark.gpu
@pytest.mark.parametrize("dim", DIMS)
def test_widths(gpu, dim):
    for post, pre in (("rms", "rms"), ("layer", "layer")):
        if dim == 1 and post == "layer":
            continue  # a single number about its mean is 0
        for rows in (1, 7):
            check(run(gpu, (rows, dim), post, pre, seed=dim), f"{post}/{pre} {rows} x {dim}")


@pytest.mark.gpu
@pytest.mark.parametrize("post", KINDS)
@pytest.mark.parametrize("pre", KINDS)
@pytest.mark.parametrize("modulated", [False, True])
@pytest.mark.parametrize("dim", [96, 1279, 2560, 17000])
def test_kinds(gpu, post, pre, modulated, dim):
    check(run(gpu, (2, 33, dim), post, pre, modulated, bias=not modulated or pre == "layer"),
          f"{post}/{pre} modulated {modulated} {dim}")


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [80, 1280, 5001, 16388])
@pytest.mark.parametrize("parts", [dict(gate=False), dict(bias=False), dict(sum=False), dict(out=False),
                                   dict(y=False), dict(y=False, sum=False), dict(gate=False, bias=False, sum=False)])
def test_parts_left_out(gpu, dim, parts):
    check(run(gpu, (3, 5, dim), **parts), f"{dim} {parts}")


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 63, 64, 255, 1000, 5000, 70000])
def test_counts_of_rows(gpu, rows):
    check(run(gpu, (rows, 64), "layer", "rms"), f"{rows} rows")
    if rows <= 5000:
        check(run(gpu, (rows, 1280), "rms", "layer"), f"{rows} rows")


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 1280, 1283, 17000])
@pytest.mark.parametrize("which", ["sum=residual", "sum=y", "out=y", "out=residual", "both"])
def test_in_place(gpu, dim, which):
    def place(y, r, s, o):
        return {"sum=residual": (y, r, r, o), "sum=y": (y, r, y, o), "out=y": (y, r, s, y),
                "out=residual": (y, r, s, r), "both": (y, r, r, y)}[which]

    check(run(gpu, (2, 21, dim), "layer", "rms", place=place), f"{which} {dim}")


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 320, 1281])
@pytest.mark.parametrize("pad", [1, 4, 100])
def test_rows_apart(gpu, dim, pad):
    """Rows further apart than they are long, and in an order of their own; what lies between is left."""
    between = []

    def place(y, r, s, o):
        def spread(t):
            buf = torch.full((21, 2, dim + pad), 7.5, device=gpu)
            view = buf[:, :, :dim].permute(1, 0, 2)
            view.copy_(t)
            between.append(buf)
            return view

        return spread(y), r, spread(s), o

    check(run(gpu, (2, 21, dim), "rms", "layer", place=place), f"{dim} + {pad}")
    assert all((b[:, :, dim:] == 7.5).all() for b in between)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [320, 1024])
def test_at_an_address_of_4(gpu, dim):
    def place(y, r, s, o):
        def shifted(t, by):
            buf = torch.full((t.numel() + 8,), float("nan"), device=gpu)
            view = buf[by:by + t.numel()].view(t.shape)
            view.copy_(t)
            return view

        return shifted(y, 1), shifted(r, 2), shifted(s, 3), shifted(o, 1)

    check(run(gpu, (2, 9, dim), "layer", "layer", place=place), f"{dim}")


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 1280, 17000])
def test_operands_of_every_broadcast(gpu, dim):
    """A weight a row (one number for it), a gate for all, a bias of the whole shape."""
    r = rng(dim)
    shape = (2, 3, 5, dim)
    y, res = normal(r, shape), normal(r, shape)
    weight, gate, bias = normal(r, (3, 5, 1), 1.0, 0.2), normal(r, (1,)), normal(r, shape)
    s, o = unwritten(shape, gpu), unwritten(shape, gpu)
    sdhip.norm_residual(dev(y, gpu), dev(res, gpu), s, o, sdhip.row_norm("rms", 1e-5, dev(weight, gpu), dev(bias, gpu)),
                        sdhip.row_norm("layer", 1e-5), dev(gate, gpu))
    z, zs = norm64("rms", y.astype(np.float64), 1e-5, weight.astype(np.float64), bias.astype(np.float64), 0.0)
    want = res + gate * z
    size = np.abs(res) + np.abs(gate) * zs
    assert (np.abs(s.cpu().numpy() - want) <= 12 * U * size).all()
    n, _ = norm64("layer", s.cpu().numpy().astype(np.float64), 1e-5, None, None, 0.0)
    assert (np.abs(o.cpu().numpy() - n) <= 10 * U * (np.abs(n) + 1e-3)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [96, 1280, 17000])
@pytest.mark.parametrize("power", [-90, 100])
def test_great_and_small_numbers(gpu, dim, power):
    """Their squares pass single precision; the norm of them does not."""
    r = rng(dim)
    shape = (3, dim)
    y = normal(r, shape) * np.float32(2.0 ** power)
    check(run(gpu, shape, "rms", "layer", eps=0.0, y_np=y), f"2^{power} {dim}")
    check(run(gpu, shape, "layer", "rms", eps=0.0, y_np=y), f"2^{power} {dim}")


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [96, 1280, 17000])
def test_far_from_zero(gpu, dim):
    """Rows whose mean is 10^5 times their spread."""
    r = rng(dim)
    check(run(gpu, (3, dim), "layer", "rms", y_np=normal(r, (3, dim), 1e5, 1.0)), f"{dim}")


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [96, 1280, 17000])
def test_infinities_and_nans_stay_in_their_rows(gpu, dim):
    r = rng(dim)
    y, res = normal(r, (6, dim)), normal(r, (6, dim))
    y[1, 5], res[4, dim - 1] = np.nan, np.inf
    s, o = unwritten((6, dim), gpu), unwritten((6, dim), gpu)
    sdhip.norm_residual(dev(y, gpu), dev(res, gpu), s, o, sdhip.row_norm("rms", 1e-6), sdhip.row_norm("layer", 1e-6))
    s, o = s.cpu().numpy(), o.cpu().numpy()
    assert np.isnan(s[1]).all() and np.isnan(o[1]).all() and np.isnan(o[4]).all()
    assert np.isinf(s[4, -1]) and np.isfinite(s[4, :-1]).all()
    keep = [0, 2, 3, 5]
    assert np.isfinite(s[keep]).all() and np.isfinite(o[keep]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 1280, 17000])
def test_captured_and_replayed(gpu, dim):
    r = rng(dim)
    shape = (2, 40, dim)
    y, res, w = dev(normal(r, shape), gpu), dev(normal(r, shape), gpu), dev(normal(r, (dim,), 1.0, 0.1), gpu)
    s, o = unwritten(shape, gpu), unwritten(shape, gpu)

    def call():
        sdhip.norm_residual(y, res, s, o, sdhip.row_norm("rms", 1e-6, w), sdhip.row_norm("layer", 1e-6, w))

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            call()
    torch.cuda.current_stream().wait_stream(side)
    for i in range(3):
        y.copy_(dev(normal(rng(70 + i), shape), gpu))
        call()
        want = s.clone(), o.clone()
        s.fill_(float("nan"))
        o.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(s, want[0]) and torch.equal(o, want[1])


@pytest.mark.gpu
def test_more_rows_than_a_launch_takes(gpu):
    """2^25 + 5 rows: a launch of 64 threads a row takes 2^25 of them."""
    rows, dim = 2 ** 25 + 5, 4
    y = torch.randn((rows, dim), device=gpu, generator=torch.Generator(gpu).manual_seed(5))
    res = torch.randn((rows, dim), device=gpu, generator=torch.Generator(gpu).manual_seed(6))
    out = torch.full_like(y, float("nan"))
    sdhip.norm_residual(y, res, None, out, sdhip.row_norm("rms", 1e-6), sdhip.row_norm("none", 0.0))
    torch.cuda.synchronize()
    for part in (slice(0, 9), slice(rows // 2, rows // 2 + 9), slice(rows - 9, rows)):
        v, r = y[part].double(), res[part].double()
        z = v * (v.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
        assert ((out[part].double() - (r + z)).abs() <= 10 * U * (z.abs() + r.abs())).all()
    assert not out.isnan().any()


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [96, 1280, 17000])
@pytest.mark.parametrize("power", [-140, -130, 126])
def test_greatest_and_least_numbers(gpu, dim, power):
    """Rows whose reciprocal root is no normal number of single precision: numbers
    of 2^power, whole multiples of 2^-149, whose RMS norm is of order 1."""
    r = rng(dim)
    shape = (3, dim)
    y = np.clip(normal(r, shape), -3.5, 3.5).astype(np.float64)
    y = (y * 2.0 ** power).astype(np.float32)
    assert np.isfinite(y).all() and (y != 0).mean() > 0.9
    check(run(gpu, shape, "rms", "layer", eps=0.0, y_np=y), f"2^{power} {dim}")
