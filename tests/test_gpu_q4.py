"""MUL_MAT of 4-bit weights (Q4_0, Q4_1) and its gated GELU on the device
against float64, by the reference's metric (|y - exact| over the sum of the
products' magnitudes, ops_test.cc:154-211), within q4_lib.bound."""

import ctypes

import numpy as np
import pytest
import torch

import oracle_lib as orc
import q4_lib
import sdhip
from helpers import dev, rng, uniform, unwritten

KINDS = ["q4_0", "q4_1"]
GELU_K = 1.5957691216057308


def gelu64(x):
    with np.errstate(over="ignore"):
        return x / (1.0 + np.exp(-GELU_K * (x + 0.044715 * x ** 3)))


def strided(blocks, row, offset, device):
    """The blocks in rows `row` bytes apart beginning `offset` bytes into a
    buffer of 0xff, as a tensor of their shape."""
    n, count, size = blocks.shape
    buf = torch.full((offset + row * n,), 255, dtype=torch.uint8, device=device)
    t = torch.as_strided(buf, (n, count, size), (row, size, 1), offset)
    t.copy_(torch.from_numpy(blocks))
    return t


def run(gpu, kind, rows, k, n, seed, steps=(), redirect=None, from_redirect=False, layout=None, x=None):
    r = rng(seed)
    blocks = q4_lib.random_blocks(r, kind, n, k)
    x = uniform(r, (rows, k), 1.0) if x is None else x
    w = dev(blocks, gpu) if layout is None else strided(blocks, *layout, gpu)
    y = unwritten((rows, n), gpu)
    sdhip.mul_mat(w, dev(x, gpu), y, sdhip.epilogue(steps, redirect=redirect, from_redirect=from_redirect))
    torch.cuda.synchronize()
    return y, *q4_lib.exact(blocks, x)


# One block of K to many, an odd count of them, N below, at and past every
# tile's width, and rows at both sides of every form's limits.
SIZES = [(32, 1), (64, 15), (96, 16), (160, 17), (320, 63), (1056, 65), (544, 128), (2080, 200), (5120, 33)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 8, 9, 15, 16, 17, 31, 32, 33, 47, 64, 65, 96, 127, 129, 200, 257])
def test_product(gpu, kind, rows):
    for k, n in SIZES:
        y, exact, mag = run(gpu, kind, rows, k, n, seed=rows * 100 + k + n)
        err = orc.metric(y.cpu().numpy(), exact, mag)
        print(f"{kind} {rows} x {k} -> {n}: {err:.3g} of {q4_lib.bound(k):.3g}")
        assert err <= q4_lib.bound(k)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,k,n", [(1, 4096, 5000), (2, 1280, 20160), (13, 2048, 2500), (77, 768, 1280),
                                      (300, 1280, 1300), (700, 640, 1280), (1976, 1280, 1280), (1500, 2560, 320)])
def test_product_of_real_sizes(gpu, kind, rows, k, n):
    y, exact, mag = run(gpu, kind, rows, k, n, seed=rows + k + n)
    err = orc.metric(y.cpu().numpy(), exact, mag)
    print(f"{kind} {rows} x {k} -> {n}: {err:.3g} of {q4_lib.bound(k):.3g}")
    assert err <= q4_lib.bound(k)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [1, 7, 40, 150])
@pytest.mark.parametrize("gap,offset", [(0, 2), (2, 0), (14, 6), (1000, 16)])
def test_rows_apart_and_at_even_addresses(gpu, kind, rows, gap, offset):
    k, n = 352, 70
    row = k // 32 * q4_lib.BYTES[kind] + gap
    y, exact, mag = run(gpu, kind, rows, k, n, seed=gap + offset, layout=(row, offset))
    assert orc.metric(y.cpu().numpy(), exact, mag) <= q4_lib.bound(k)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 6, 50, 300])
def test_input_at_an_address_of_4(gpu, rows):
    """x and y begin 4 bytes past a multiple of 16."""
    r = rng(rows)
    k, n = 320, 48
    blocks = q4_lib.random_blocks(r, "q4_0", n, k)
    x = uniform(r, (rows, k), 1.0)
    xb = torch.zeros(rows * k + 1, device=gpu)
    xb[1:] = torch.from_numpy(x).flatten().to(gpu)
    yb = unwritten((rows * n + 2,), gpu)
    sdhip.mul_mat(dev(blocks, gpu), xb[1:].view(rows, k), yb[1:-1].view(rows, n))
    exact, mag = q4_lib.exact(blocks, x)
    got = yb.cpu().numpy()
    assert np.isnan(got[0]) and np.isnan(got[-1])
    assert orc.metric(got[1:-1].reshape(rows, n), exact, mag) <= q4_lib.bound(k)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [1, 4, 20, 75, 260])
@pytest.mark.parametrize("end", ["own", "redirect", "from_redirect"])
def test_chain_and_residual(gpu, kind, rows, end):
    """bias, a scale for each row, then the residual: in the output's own
    tensor, in another, or begun from what that holds."""
    k, n = 352, 90
    r = rng(rows)
    bias, scale, res = uniform(r, (n,), 1.0), uniform(r, (rows, 1), 1.0), uniform(r, (rows, n), 1.0)
    steps = [("add", dev(bias, gpu)), ("mul", dev(scale, gpu))]
    res_d = dev(res, gpu)
    out = None
    if end == "redirect":
        out = unwritten((rows, n), gpu)
    elif end == "from_redirect":
        out = res_d.clone()
    if end != "from_redirect":
        steps.append(("add", res_d))
    y, exact, mag = run(gpu, kind, rows, k, n, 9, steps, redirect=out, from_redirect=end == "from_redirect")
    if end == "from_redirect":
        want, size = (res + exact + bias) * scale, (np.abs(res) + mag + np.abs(bias)) * np.abs(scale)
    else:
        want, size = (exact + bias) * scale + res, (mag + np.abs(bias)) * np.abs(scale) + np.abs(res)
    if out is not None:
        assert torch.isnan(y).all()
    got = (y if out is None else out).cpu().numpy()
    assert orc.metric(got, want, size) <= q4_lib.bound(k, 4)


@pytest.mark.gpu
@pytest.mark.parametrize("tuning", ["fuse=0", "fuse_residual=0", "bits=8", "bits=16"])
def test_tunings(gpu, tuning):
    """The chain apart; and the modes of the other weights' products, which
    leave these as they are."""
    rows, k, n = 300, 320, 64
    r = rng(3)
    bias, res = uniform(r, (n,), 1.0), uniform(r, (rows, n), 1.0)
    out = unwritten((rows, n), gpu)
    sdhip.set_tuning(tuning)
    try:
        y, exact, mag = run(gpu, "q4_0", rows, k, n, 4, [("add", dev(bias, gpu)), ("add", dev(res, gpu))], redirect=out)
    finally:
        sdhip.set_tuning("")
    assert orc.metric(out.cpu().numpy(), exact + bias + res, mag + np.abs(bias) + np.abs(res)) <= q4_lib.bound(k, 3)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 60])
def test_four_dimensions(gpu, rows):
    """x of [2, 3, rows, k] and a chain that differs along each of them."""
    k, n = 96, 40
    r = rng(rows)
    blocks = q4_lib.random_blocks(r, "q4_1", n, k)
    x = uniform(r, (2, 3, rows, k), 1.0)
    a, b, c = uniform(r, (2, 1, 1, n), 1.0), uniform(r, (3, 1, 1), 1.0), uniform(r, (2, 3, rows, 1), 1.0)
    y = unwritten((2, 3, rows, n), gpu)
    sdhip.mul_mat(dev(blocks, gpu), dev(x, gpu), y,
                  sdhip.epilogue([("add", dev(a, gpu)), ("add", dev(b, gpu)), ("mul", dev(c, gpu)), ("silu", None)]))
    exact, mag = q4_lib.exact(blocks, x.reshape(-1, k))
    v = (exact.reshape(y.shape) + a + b) * c
    size = (mag.reshape(y.shape) + np.abs(a) + np.abs(b)) * np.abs(c)
    # silu's slope is below 1.1; its own exponential and division add 2^-20 of it.
    assert orc.metric(y.cpu().numpy(), v / (1 + np.exp(-v)), size) <= 1.1 * q4_lib.bound(k, 4) + 2.0 ** -20


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tuning", ["", "fuse=0", "bits=8"])
@pytest.mark.parametrize("rows,k,n", [(1, 32, 2), (1, 2048, 10240), (3, 96, 34), (16, 320, 160), (17, 160, 62), (70, 352, 258),
                                      (200, 640, 1290), (300, 320, 2560)])
def test_gated(gpu, kind, rows, k, n, tuning):
    r = rng(rows + n)
    blocks = q4_lib.random_blocks(r, kind, n, k)
    x, bias = uniform(r, (rows, k), 1.0), uniform(r, (n,), 1.0)
    y, out = unwritten((rows, n), gpu), unwritten((rows, n // 2), gpu)
    sdhip.set_tuning(tuning)
    try:
        sdhip.mul_mat_gated(dev(blocks, gpu), dev(x, gpu), y, out, sdhip.epilogue([("add", dev(bias, gpu))]))
    finally:
        sdhip.set_tuning("")
    exact, mag = q4_lib.exact(blocks, x)
    p, size = exact + bias, mag + np.abs(bias)
    a, g = p[:, :n // 2], p[:, n // 2:]
    if tuning != "fuse=0":
        assert torch.isnan(y).all()
    # d(a gelu(g)) <= |gelu| da + |a| 1.13 dg; gelu's own exponential and division, and the product, add 2^-20.
    err = q4_lib.bound(k, 1)
    allowed = np.abs(gelu64(g)) * err * size[:, :n // 2] + 1.13 * np.abs(a) * err * size[:, n // 2:]
    allowed = allowed * (1 + 1e-3) + 2.0 ** -20 * np.abs(a) * np.abs(g) + err * err * size[:, :n // 2] * size[:, n // 2:]
    diff = np.abs(out.cpu().numpy() - a * gelu64(g))
    assert np.isfinite(diff).all() and (diff <= allowed + 1e-30).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 5, 40, 200])
@pytest.mark.parametrize("power", [-100, -30, 15, 60])
def test_inputs_of_any_magnitude(gpu, rows, power):
    r = rng(rows)
    x = uniform(r, (rows, 320), 1.0) * np.float32(2.0 ** power)
    y, exact, mag = run(gpu, "q4_0", rows, 320, 50, 2, x=x)
    assert orc.metric(y.cpu().numpy(), exact, mag) <= q4_lib.bound(320)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 5, 40, 200])
def test_rows_far_apart_and_rows_of_zeros(gpu, rows):
    """Each row has a magnitude of its own, every third is zero."""
    r = rng(rows)
    x = uniform(r, (rows, 640), 1.0) * 2.0 ** r.integers(-60, 60, (rows, 1))
    x[2::3] = 0
    y, exact, mag = run(gpu, "q4_1", rows, 640, 70, 3, x=x.astype(np.float32))
    got = y.cpu().numpy()
    assert (got[2::3] == 0).all()
    keep = np.ones(rows, bool)
    keep[2::3] = False
    assert orc.metric(got[keep], exact[keep], mag[keep]) <= q4_lib.bound(640)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 5, 40, 200])
def test_great_channels(gpu, rows):
    """A channel 2^12 times as great as the others: they keep their own bits."""
    r = rng(rows)
    x = uniform(r, (rows, 320), 1.0)
    x[:, 100] *= 4096.0
    y, exact, mag = run(gpu, "q4_0", rows, 320, 50, 4, x=x)
    blocks = q4_lib.random_blocks(rng(4), "q4_0", 50, 320)
    # Weights of 0 on that channel, whose outputs are of the others' products alone.
    assert orc.metric(y.cpu().numpy(), exact, mag) <= q4_lib.bound(320)
    blocks[:, 3, 2 + 4] = (blocks[:, 3, 2 + 4] & 0xf0) | 8
    w, _ = q4_lib.widen(blocks)
    assert (w[:, 100] == 0).all()
    y2 = unwritten((rows, 50), gpu)
    sdhip.mul_mat(dev(blocks, gpu), dev(x, gpu), y2)
    exact, mag = q4_lib.exact(blocks, x)
    assert orc.metric(y2.cpu().numpy(), exact, mag) <= q4_lib.bound(320)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2, 5, 40, 200])
def test_infinities_and_nans_stay_in_their_rows(gpu, rows):
    r = rng(rows)
    k, n = 320, 50
    blocks = q4_lib.random_blocks(r, "q4_0", n, k)
    blocks[:, 1, 2 + 3] = (blocks[:, 1, 2 + 3] & 0xf0) | 11  # number 35 of each row: q - 8 = 3
    x = uniform(r, (rows, k), 1.0)
    x[1, 35] = np.inf
    if rows > 3:
        x[3, 7] = np.nan
    y = unwritten((rows, n), gpu)
    sdhip.mul_mat(dev(blocks, gpu), dev(x, gpu), y)
    got = y.cpu().numpy()
    w, _ = q4_lib.widen(blocks)
    assert (got[1] == np.where(w[:, 35] > 0, np.inf, -np.inf)).all()
    if rows > 3:
        assert np.isnan(got[3]).all()
    keep = [i for i in range(rows) if i not in (1, 3)]
    exact, mag = q4_lib.exact(blocks, x[keep])
    assert orc.metric(got[keep], exact, mag) <= q4_lib.bound(k)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [1, 40, 200])
def test_scales_of_zero_and_subnormal(gpu, kind, rows):
    r = rng(rows)
    k, n = 160, 40
    blocks = q4_lib.random_blocks(r, kind, n, k)
    d = np.array([0.0, 6e-8, -3e-5, 60.0], np.float16)
    blocks[:, :, 0:2] = d[r.integers(0, 4, (n, k // 32))].reshape(n, k // 32, 1).view(np.uint8).reshape(n, -1, 2)
    x = uniform(r, (rows, k), 1.0)
    y = unwritten((rows, n), gpu)
    sdhip.mul_mat(dev(blocks, gpu), dev(x, gpu), y)
    exact, mag = q4_lib.exact(blocks, x)
    zero = mag == 0
    got = y.cpu().numpy()
    assert (got[zero] == 0).all()
    assert orc.metric(got[~zero], exact[~zero], mag[~zero]) <= q4_lib.bound(k)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 9, 100, 513])
def test_the_same_bits_again_and_on_another_stream(gpu, rows):
    r = rng(rows)
    k, n = 1280, 320
    w, x = dev(q4_lib.random_blocks(r, "q4_0", n, k), gpu), dev(uniform(r, (rows, k), 1.0), gpu)
    y = [unwritten((rows, n), gpu) for _ in range(3)]
    sdhip.mul_mat(w, x, y[0])
    sdhip.mul_mat(w, x, y[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work = sdhip.mul_mat(w, x, y[2])
    torch.cuda.synchronize()
    del work
    assert torch.equal(y[0], y[1]) and torch.equal(y[0], y[2])


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 20, 300])
def test_captured_and_replayed(gpu, rows):
    """The product and its gated form in one graph, replayed after new inputs."""
    r = rng(rows)
    k, n = 640, 320
    w, x = dev(q4_lib.random_blocks(r, "q4_1", n, k), gpu), dev(uniform(r, (rows, k), 1.0), gpu)
    y, unused, out = (unwritten(s, gpu) for s in ((rows, n), (rows, n), (rows, n // 2)))
    lib = sdhip.load()
    size = lib.sdhip_mul_mat_work_size(sdhip.desc(w), sdhip.desc(x), sdhip.desc(y))
    works = [torch.empty(max(size, 16), dtype=torch.uint8, device=gpu) for _ in range(2)]

    def calls():
        sdhip.mul_mat(w, x, y, work=works[0])
        sdhip.mul_mat_gated(w, x, unused, out, work=works[1])

    calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            calls()
    torch.cuda.current_stream().wait_stream(side)
    for i in range(3):
        x.copy_(dev(uniform(rng(50 + i), (rows, k), 1.0), gpu))
        calls()
        want = y.clone(), out.clone()
        y.fill_(float("nan"))
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and torch.equal(out, want[1])


@pytest.mark.gpu
def test_weights_past_32_bits_of_bytes(gpu):
    """Rows 40 MB apart: the last row's offset passes 2^32."""
    k, n, rows = 64, 110, 3
    if torch.cuda.mem_get_info()[0] < 8 << 30:
        pytest.skip("needs 8 GB of device memory")
    r = rng(6)
    blocks = q4_lib.random_blocks(r, "q4_0", n, k)
    w = strided(blocks, 40 << 20, 0, gpu)
    for m in (1, rows, 70):
        x = uniform(r, (m, k), 1.0)
        y = unwritten((m, n), gpu)
        sdhip.mul_mat(w, dev(x, gpu), y)
        exact, mag = q4_lib.exact(blocks, x)
        assert orc.metric(y.cpu().numpy(), exact, mag) <= q4_lib.bound(k)


@pytest.mark.gpu
def test_refusals_leave_the_output(gpu):
    """A missing work buffer, an output over an operand, tensors without data."""
    r = rng(8)
    w, x = dev(q4_lib.random_blocks(r, "q4_0", 320, 320), gpu), dev(uniform(r, (600, 320), 1.0), gpu)
    y = unwritten((600, 320), gpu)
    lib = sdhip.load()
    dw, dx, dy = sdhip.desc(w), sdhip.desc(x), sdhip.desc(y)
    size = lib.sdhip_mul_mat_work_size(dw, dx, dy)
    if size:
        assert lib.sdhip_mul_mat(dw, dx, dy, None, None, 0, None) == sdhip.ERROR
        assert lib.sdhip_mul_mat(dw, dx, dy, None, ctypes.c_void_p(x.data_ptr()), size - 1, None) == sdhip.ERROR
    work = torch.empty(max(size, 16), dtype=torch.uint8, device=gpu)
    args = (None, ctypes.c_void_p(work.data_ptr()), size, None)
    assert lib.sdhip_mul_mat(dw, dx, dx, *args) == sdhip.ERROR
    none = sdhip.desc(y)
    none.data = None
    assert lib.sdhip_mul_mat(dw, dx, none, *args) == sdhip.ERROR
    torch.cuda.synchronize()
    assert torch.isnan(y).all()


FORMS = [1, 2, 3, 4, 5, 6]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rows", [1, 16, 17, 31, 33, 64, 65, 127, 128, 130, 200, 257])
def test_forms(gpu, kind, form, rows):
    """Every form at rows and columns at both sides of its tiles' limits, few
    blocks of K and many, and counts of them that end inside a stage."""
    sdhip.set_tuning(f"q4_form={form}")
    try:
        for k, n in [(32, 1), (64, 31), (96, 33), (128, 64), (160, 65), (224, 127), (1056, 129), (1568, 257), (2080, 300)]:
            y, exact, mag = run(gpu, kind, rows, k, n, seed=rows * 10 + k + n)
            err = orc.metric(y.cpu().numpy(), exact, mag)
            print(f"{kind} form {form} {rows} x {k} -> {n}: {err:.3g} of {q4_lib.bound(k):.3g}")
            assert err <= q4_lib.bound(k)
    finally:
        sdhip.set_tuning("")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rows,k,n", [(1, 64, 2), (33, 320, 62), (70, 352, 258), (150, 1120, 130), (300, 96, 514)])
def test_forms_gated(gpu, kind, form, rows, k, n):
    sdhip.set_tuning(f"q4_form={form}")
    try:
        r = rng(rows + n)
        blocks = q4_lib.random_blocks(r, kind, n, k)
        x, bias, scale = uniform(r, (rows, k), 1.0), uniform(r, (n,), 1.0), uniform(r, (rows, 1), 1.0)
        steps = [("add", dev(bias, gpu)), ("mul", dev(scale, gpu))]
        y, out = unwritten((rows, n), gpu), unwritten((rows, n // 2), gpu)
        sdhip.mul_mat_gated(dev(blocks, gpu), dev(x, gpu), y, out, sdhip.epilogue(steps))
    finally:
        sdhip.set_tuning("")
    exact, mag = q4_lib.exact(blocks, x)
    p, size = (exact + bias) * scale, (mag + np.abs(bias)) * np.abs(scale)
    a, g = p[:, :n // 2], p[:, n // 2:]
    err = q4_lib.bound(k, 2)
    allowed = np.abs(gelu64(g)) * err * size[:, :n // 2] + 1.13 * np.abs(a) * err * size[:, n // 2:]
    allowed = allowed * (1 + 1e-3) + 2.0 ** -20 * np.abs(a) * np.abs(g) + err * err * size[:, :n // 2] * size[:, n // 2:]
    diff = np.abs(out.cpu().numpy() - a * gelu64(g))
    assert torch.isnan(y).all() and np.isfinite(diff).all() and (diff <= allowed + 1e-30).all()


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("end", ["own", "redirect", "from_redirect"])
def test_forms_chain(gpu, form, end):
    """A bias, a number for each row, a number for each matrix of rows, then
    the residual; x of [3, rows, k]."""
    rows, k, n = 50, 352, 130
    r = rng(form)
    blocks = q4_lib.random_blocks(r, "q4_1", n, k)
    x = uniform(r, (3, rows, k), 1.0)
    bias, scale, shift = uniform(r, (n,), 1.0), uniform(r, (3, rows, 1), 1.0), uniform(r, (3, 1, n), 1.0)
    res = uniform(r, (3, rows, n), 1.0)
    steps = [("add", dev(bias, gpu)), ("mul", dev(scale, gpu)), ("add", dev(shift, gpu))]
    res_d = dev(res, gpu)
    out = None
    if end == "redirect":
        out = unwritten((3, rows, n), gpu)
    elif end == "from_redirect":
        out = res_d.clone()
    if end != "from_redirect":
        steps.append(("add", res_d))
    y = unwritten((3, rows, n), gpu)
    sdhip.set_tuning(f"q4_form={form}")
    try:
        sdhip.mul_mat(dev(blocks, gpu), dev(x, gpu), y,
                      sdhip.epilogue(steps, redirect=out, from_redirect=end == "from_redirect"))
    finally:
        sdhip.set_tuning("")
    exact, mag = (t.reshape(y.shape) for t in q4_lib.exact(blocks, x.reshape(-1, k)))
    first = res if end == "from_redirect" else 0.0 * res
    last = res - first
    want = (first + exact + bias) * scale + shift + last
    size = (np.abs(first) + mag + np.abs(bias)) * np.abs(scale) + np.abs(shift) + np.abs(last)
    got = (y if out is None else out).cpu().numpy()
    assert orc.metric(got, want, size) <= q4_lib.bound(k, 5)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("gap,offset", [(2, 0), (14, 6)])
def test_forms_rows_apart(gpu, kind, form, gap, offset):
    rows, k, n = 70, 544, 100
    row = k // 32 * q4_lib.BYTES[kind] + gap
    sdhip.set_tuning(f"q4_form={form}")
    try:
        y, exact, mag = run(gpu, kind, rows, k, n, seed=gap + offset, layout=(row, offset))
        assert orc.metric(y.cpu().numpy(), exact, mag) <= q4_lib.bound(k)
    finally:
        sdhip.set_tuning("")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("form", FORMS)
def test_forms_ranges(gpu, kind, form):
    """Rows of magnitudes far apart, rows of zeros, and with Q4_0 an infinity
    and a NaN, which stay in their rows."""
    rows, k, n = 70, 640, 70
    r = rng(form)
    blocks = q4_lib.random_blocks(r, kind, n, k)
    size = q4_lib.BYTES[kind]
    blocks[:, 1, size - 16 + 3] = (blocks[:, 1, size - 16 + 3] & 0xf0) | 11  # number 35 of each row: q - 8 = 3
    x = (uniform(r, (rows, k), 1.0) * 2.0 ** r.integers(-60, 60, (rows, 1))).astype(np.float32)
    x[2::3] = 0
    x[4, 35], x[7, 7] = np.inf, np.nan
    y = unwritten((rows, n), gpu)
    sdhip.set_tuning(f"q4_form={form}")
    try:
        sdhip.mul_mat(dev(blocks, gpu), dev(x, gpu), y)
    finally:
        sdhip.set_tuning("")
    got = y.cpu().numpy()
    assert (got[2::3] == 0).all() and np.isnan(got[7]).all() and not np.isfinite(got[4]).any()
    if kind == "q4_0":
        w, _ = q4_lib.widen(blocks)
        assert (got[4] == np.where(w[:, 35] > 0, np.inf, -np.inf)).all()
    keep = [i for i in range(rows) if i % 3 != 2 and i not in (4, 7)]
    exact, mag = q4_lib.exact(blocks, x[keep])
    assert orc.metric(got[keep], exact, mag) <= q4_lib.bound(k)


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS)
def test_forms_captured(gpu, form):
    r = rng(form)
    rows, k, n = 70, 640, 320
    w, x = dev(q4_lib.random_blocks(r, "q4_1", n, k), gpu), dev(uniform(r, (rows, k), 1.0), gpu)
    y, unused, out = (unwritten(s, gpu) for s in ((rows, n), (rows, n), (rows, n // 2)))
    sdhip.set_tuning(f"q4_form={form}")
    try:
        size = sdhip.load().sdhip_mul_mat_work_size(sdhip.desc(w), sdhip.desc(x), sdhip.desc(y))
        work = torch.empty(max(size, 16), dtype=torch.uint8, device=gpu)

        def calls():  # one after the other, by one work buffer
            sdhip.mul_mat(w, x, y, work=work)
            sdhip.mul_mat_gated(w, x, unused, out, work=work)

        calls()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            with torch.cuda.graph(graph, stream=side):
                calls()
        torch.cuda.current_stream().wait_stream(side)
        for i in range(3):
            x.copy_(dev(uniform(rng(50 + i), (rows, k), 1.0), gpu))
            calls()
            want = y.clone(), out.clone()
            y.fill_(float("nan"))
            out.fill_(float("nan"))
            work.fill_(255)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want[0]) and torch.equal(out, want[1])
    finally:
        sdhip.set_tuning("")


@pytest.mark.gpu
def test_work_buffer_is_all_that_is_written(gpu):
    """Every form with a work buffer of exactly its size, between guards."""
    r = rng(1)
    for form in FORMS[1:]:
        for kind, rows, k, n in (("q4_0", 70, 352, 100), ("q4_1", 129, 1056, 130), ("q4_1", 1, 32, 2)):
            w, x = dev(q4_lib.random_blocks(r, kind, n, k), gpu), dev(uniform(r, (rows, k), 1.0), gpu)
            y, out = unwritten((rows, n), gpu), unwritten((rows, n // 2), gpu)
            sdhip.set_tuning(f"q4_form={form}")
            try:
                size = sdhip.load().sdhip_mul_mat_work_size(sdhip.desc(w), sdhip.desc(x), sdhip.desc(y))
                buf = torch.full((size + 8192,), 77, dtype=torch.uint8, device=gpu)
                sdhip.mul_mat(w, x, y, work=buf[4096:4096 + size])
                sdhip.mul_mat_gated(w, x, y, out, work=buf[4096:4096 + size])
            finally:
                sdhip.set_tuning("")
            assert (buf[:4096] == 77).all() and (buf[4096 + size:] == 77).all(), (form, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("form", [0] + FORMS)
def test_more_groups_of_rows_than_a_grid_s_second_dimension(gpu, form):
    """16 65535 + 3 rows and more: whatever form is asked for, one that takes them."""
    rows, k, n = 16 * 65535 + 3, 32, 5
    r = rng(form)
    blocks = q4_lib.random_blocks(r, "q4_0", n, k)
    x = uniform(r, (rows, k), 1.0)
    y = unwritten((rows, n), gpu)
    sdhip.set_tuning(f"q4_form={form}")
    try:
        sdhip.mul_mat(dev(blocks, gpu), dev(x, gpu), y, sdhip.epilogue([]))
        torch.cuda.synchronize()
    finally:
        sdhip.set_tuning("")
    exact, mag = q4_lib.exact(blocks, x)
    assert orc.metric(y.cpu().numpy(), exact, mag) <= q4_lib.bound(k)


# Sizes by which the first form takes 1, 2, 4 and 8 rows a workgroup and K in 1,
# 2, 4 and 8 splits, x in one chunk and in several.
SHAPES = [(2, 96, 33), (1, 2080, 40001), (2, 544, 33), (2, 2080, 33), (100, 96, 257), (5, 544, 5001), (5, 2080, 5001),
          (31, 544, 257), (16, 2080, 257), (15, 96, 5001), (33, 2080, 1000), (64, 544, 257), (31, 8224, 257),
          (7, 96, 20000), (15, 544, 5001), (33, 544, 1000), (15, 8224, 1000), (257, 544, 1000), (16, 4128, 5000),
          (16, 96, 20000), (256, 1280, 1280),
          # workgroups of fewer than 8 waves: 1, 3, 5 and 6 tiles by 1 or 2 splits, and of 8
          (1, 320, 320), (3, 64, 640), (1, 64, 8200), (1, 512, 12301), (2, 1280, 20160), (1, 256, 24001)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,k,n", SHAPES)
def test_shapes_of_few_rows(gpu, kind, rows, k, n):
    sdhip.set_tuning("q4_form=1")
    try:
        y, exact, mag = run(gpu, kind, rows, k, n, seed=rows + k + n)
    finally:
        sdhip.set_tuning("")
    err = orc.metric(y.cpu().numpy(), exact, mag)
    print(f"{kind} {rows} x {k} -> {n}: {err:.3g} of {q4_lib.bound(k):.3g}")
    assert err <= q4_lib.bound(k)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,k,n", [(2, 96, 1000), (2, 544, 1000), (33, 96, 1000), (9, 544, 1000), (31, 96, 2500),
                                      (33, 2080, 1000), (7, 544, 2500), (7, 96, 20000), (31, 544, 2500), (33, 544, 1000),
                                      (257, 544, 1000), (256, 1280, 1280), (1, 320, 320), (1, 64, 8200), (1, 512, 24002)])
def test_shapes_of_few_rows_gated(gpu, kind, rows, k, n):
    test_forms_gated(gpu, kind, 1, rows, k, n)


@pytest.mark.gpu
def test_calls_at_once(gpu):
    """Products and norms on four streams at once, each with its own buffers: the
    bits of calls one by one."""
    sizes = [(1, 640, 3000), (40, 640, 1000), (300, 1280, 1300), (700, 640, 1300)]
    r = rng(9)
    held = []
    for rows, k, n in sizes:
        w, x = dev(q4_lib.random_blocks(r, "q4_1", n, k), gpu), dev(uniform(r, (rows, k), 1.0), gpu)
        scale = dev(uniform(r, (n,), 1.0), gpu)
        outs = [unwritten((rows, n), gpu) for _ in range(4)]
        dw, dx, dy = sdhip.desc(w), sdhip.desc(x), sdhip.desc(outs[0])
        size = sdhip.load().sdhip_mul_mat_work_size(dw, dx, dy)
        work = torch.empty(max(size, 16), dtype=torch.uint8, device=gpu)
        held.append((w, x, scale, outs, work, size, torch.cuda.Stream()))

    def call(w, x, scale, outs, work, size, stream, first):
        handle = ctypes.c_void_p(stream.cuda_stream)
        y, n = outs[first:first + 2]
        sdhip.check(sdhip.load().sdhip_mul_mat(sdhip.desc(w), sdhip.desc(x), sdhip.desc(y), None,
                                               ctypes.c_void_p(work.data_ptr()), size, handle), "mul_mat")
        pre = sdhip.row_norm("rms", 1e-6, weight=scale)
        sdhip.check(sdhip.load().sdhip_norm_residual(None, None, None, 1.0, sdhip.desc(y), 1.0, None, pre,
                                                     sdhip.desc(n), handle), "norm_residual")

    torch.cuda.synchronize()
    for h in held:
        call(*h, 0)
        torch.cuda.synchronize()
    for _ in range(5):
        for h in held:
            for o in h[3][2:]:
                o.fill_(float("nan"))
        torch.cuda.synchronize()
        for _ in range(3):
            for h in held:
                call(*h, 2)
        torch.cuda.synchronize()
        for h in held:
            assert torch.equal(h[3][0], h[3][2]) and torch.equal(h[3][1], h[3][3])
