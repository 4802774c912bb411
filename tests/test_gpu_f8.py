"""MUL_MAT of E4M3 weights with block scales and its gated GELU on the device
against float64, by the reference's metric (|y - exact| over the sum of the
products' magnitudes, ops_test.cc:154-211), within f8_lib.bound."""

import ctypes

import numpy as np
import pytest
import torch

import f8_lib
import oracle_lib as orc
import sdhip
from helpers import dev, rng, uniform, unwritten

GELU_K = 1.5957691216057308


def gelu64(x):
    with np.errstate(over="ignore"):
        return x / (1.0 + np.exp(-GELU_K * (x + 0.044715 * x ** 3)))


def weights(w, device, row=None, offset=0):
    """The bytes as float8 on the device, rows `row` bytes apart from `offset` on
    in a buffer of NaN."""
    n, k = w.shape
    row = k if row is None else row
    buf = torch.full((offset + row * n,), 127, dtype=torch.uint8, device=device)
    t = torch.as_strided(buf, (n, k), (row, 1), offset)
    t.copy_(torch.from_numpy(w))
    return t.view(torch.float8_e4m3fn)


def scales_of(scales, device, apart=0):
    """The scales on the device, rows `apart` numbers past their end apart, NaN between."""
    n, b = scales.shape
    buf = torch.full((n, b + apart), float("nan"), device=device)
    buf[:, :b] = dev(scales, device)
    return buf[:, :b]


class Guarded:
    """An output with numbers before and behind it that stay as they were."""

    def __init__(self, shape, device, room=512):
        self.n = int(np.prod(shape))
        self.buf = torch.full((self.n + 2 * room,), -7.25, device=device)
        self.buf[room:room + self.n] = float("nan")
        self.t = self.buf[room:room + self.n].view(shape)
        self.room = room

    def check(self):
        assert (self.buf[:self.room] == -7.25).all() and (self.buf[self.room + self.n:] == -7.25).all()
        return self.t.cpu().numpy()


def run(gpu, rows, k, n, seed, steps=(), layout=(None, 0), x=None, apart=0, w=None):
    r = rng(seed)
    bytes_, scales = f8_lib.random_weights(r, n, k)
    bytes_ = bytes_ if w is None else w
    x = uniform(r, (rows, k), 1.0) if x is None else x
    y = Guarded((rows, n), gpu)
    sdhip.mul_mat_f8(weights(bytes_, gpu, *layout), scales_of(scales, gpu, apart), dev(x, gpu), y.t, sdhip.epilogue(steps))
    torch.cuda.synchronize()
    return y.check(), *f8_lib.exact(bytes_, scales, x)


FORMS = [0, 1, 2, 3, 4, 5, 6]


@pytest.fixture(params=FORMS)
def form(request, gpu):
    """Each form of the products in turn, whatever the size; 0 the library's choice."""
    if request.param:
        sdhip.set_tuning(f"f8_form={request.param}")
    yield request.param
    sdhip.set_tuning("")


# One number of K to many blocks, whole and not; N below, at and past every
# tile's width and a scale's block.
SIZES = [(1, 1), (16, 15), (31, 16), (100, 17), (128, 63), (129, 65), (256, 128), (320, 129), (1000, 200), (2080, 300), (5120, 33)]
ROWS = [1, 2, 3, 4, 5, 8, 15, 16, 17, 31, 32, 33, 64, 65, 96, 127, 128, 129, 200, 257]


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
def test_product(gpu, form, rows):
    for k, n in SIZES:
        y, exact, mag = run(gpu, rows, k, n, seed=rows * 100 + k + n)
        err = orc.metric(y, exact, mag)
        print(f"{rows} x {k} -> {n}: {err:.3g} of {f8_lib.bound(k):.3g}", flush=True)
        assert err <= f8_lib.bound(k)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,n", [(1, 4096, 5000), (2, 1280, 20160), (13, 2048, 2500), (77, 768, 1280), (300, 1280, 1300),
                                      (700, 640, 1280), (1976, 1280, 1280), (1500, 2560, 320)])
def test_product_of_real_sizes(gpu, rows, k, n):
    y, exact, mag = run(gpu, rows, k, n, seed=rows + k + n)
    err = orc.metric(y, exact, mag)
    print(f"{rows} x {k} -> {n}: {err:.3g} of {f8_lib.bound(k):.3g}")
    assert err <= f8_lib.bound(k)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 16, 40, 130, 300])
@pytest.mark.parametrize("k,row,offset", [(128, 128, 1), (128, 144, 8), (128, 129, 0), (320, 323, 5), (256, 272, 16), (200, 208, 0),
                                          (384, 384, 4), (1, 7, 3), (130, 131, 15)])
def test_weights_anywhere(gpu, form, rows, k, row, offset):
    """Rows of the weights at any address, NaN between and behind them."""
    y, exact, mag = run(gpu, rows, k, 150, seed=rows + k + row, layout=(row, offset), apart=3)
    assert orc.metric(y, exact, mag) <= f8_lib.bound(k)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 17, 150])
def test_every_weight(gpu, form, rows):
    """All numbers of E4M3, each found by a row of x that is one number."""
    values = [b for b in range(256) if b & 127 != 127]
    w = np.array(values, dtype=np.uint8).repeat(128).reshape(len(values), 128)
    w = np.ascontiguousarray(w.T)  # [n = 128, k = 254]
    x = np.zeros((rows, len(values)), np.float32)
    at = rng(rows).integers(0, len(values), rows)
    x[np.arange(rows), at] = 2.0
    y = Guarded((rows, 128), gpu)
    sdhip.mul_mat_f8(weights(w, gpu), torch.full((1, 2), 0.5, device=gpu), dev(x, gpu), y.t)
    torch.cuda.synchronize()
    assert (y.check() == f8_lib.TABLE[w[:, at]].T).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 16, 17, 150])
def test_numbers_of_x_are_held_as_documented(gpu, form, rows):
    """Products by 1 of one number of x each: what x's numbers are held to, bit for
    bit -- ties, both sides of 448 2^e, the least numbers, great and small groups."""
    k = 256
    r = rng(rows)
    x = np.empty((rows, k), np.float32)
    for m in range(rows):
        for b in range(2):
            top = np.float32([448, 449, 224.1, 1, 0.9, 240, 255, 447.99][(m + b) % 8] * 2.0 ** r.integers(-100, 100))
            g = (r.uniform(-1, 1, 128) * 2.0 ** r.integers(-20, 1, 128)).astype(np.float32) * top
            ties = (np.rint(r.uniform(8, 16, 128)) + 0.5) * 2.0 ** r.integers(-12, 1, 128) * top / 32
            g = np.where(r.random(128) < 0.3, ties, g)
            g[r.integers(0, 128)] = top
            x[m, 128 * b:128 * b + 128] = np.clip(g, -top, top)
    w = np.zeros((k, k), np.uint8)
    w[np.arange(k), np.arange(k)] = 0x38  # 1
    y = Guarded((rows, k), gpu)
    sdhip.mul_mat_f8(weights(w, gpu), torch.ones((2, 2), device=gpu), dev(x, gpu), y.t)
    torch.cuda.synchronize()
    want = f8_lib.held(x)
    assert (y.check() == want.astype(np.float32)).all()
    # Half a step: 2^-4 of a number, and 2^-10 2^e below 2^-6 2^e, where 224 2^e is
    # below the greatest or e is -101.
    least = np.maximum(np.abs(x).reshape(rows, 2, 128).max(-1).repeat(128, 1) * 2.0 ** -17, 2.0 ** -111)
    assert (np.abs(want - x) <= np.maximum(np.abs(x) * 2.0 ** -4, least)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 16, 17, 150])
def test_extreme_rows(gpu, form, rows):
    """Rows of single precision's greatest numbers and of small ones, of zeros, and
    of both in one row: finite wherever the sums of the products' magnitudes are."""
    k, n = 640, 70
    r = rng(rows)
    x = uniform(r, (rows, k), 1.0)
    power = np.array([127, 120, 60, 0, -60, -80, -90])[np.arange(rows) % 7]
    x = (x * 2.0 ** power[:, None]).astype(np.float32)
    x[:, 128:256] *= np.float32(2.0 ** -20)
    if rows > 3:
        x[3] = 0.0
        x[2, 300:400] = -0.0
    bytes_, scales = f8_lib.random_weights(r, n, k, scale=0.001)
    y = Guarded((rows, n), gpu)
    sdhip.mul_mat_f8(weights(bytes_, gpu), dev(scales, gpu), dev(x, gpu), y.t)
    torch.cuda.synchronize()
    exact, mag = f8_lib.exact(bytes_, scales, x)
    assert mag.max() < 2.0 ** 127
    # A sum's last bit is 2^-149, of each of the additions.
    assert (np.abs(y.check() - exact) <= f8_lib.bound(k) * mag + 140 * 2.0 ** -149).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 16, 17, 150])
def test_infinities_and_nans(gpu, form, rows):
    """An infinity or NaN in x reaches its own row, a NaN among the weights its own
    column, whatever stands against it; a scale its block."""
    k, n = 400, 140
    r = rng(rows)
    x = uniform(r, (rows, k), 1.0)
    bad = np.zeros(rows, bool)
    for m in range(0, rows, 3):
        x[m, r.integers(0, k)] = [np.inf, -np.inf, np.nan][m // 3 % 3]
        bad[m] = True
    bytes_, scales = f8_lib.random_weights(r, n, k)
    bytes_[:, :] = np.where(r.random((n, k)) < 0.2, 0, bytes_)
    bytes_[11, 333] = 127
    bytes_[129, 0] = 255
    y = Guarded((rows, n), gpu)
    sdhip.mul_mat_f8(weights(bytes_, gpu), dev(scales, gpu), dev(x, gpu), y.t)
    torch.cuda.synchronize()
    got = y.check()
    nan = bad[:, None] | np.isin(np.arange(n), (11, 129))[None]
    assert (np.isnan(got) == nan).all()
    clean = np.where(bad[:, None], 0, x), np.where((bytes_ & 127) == 127, 0, bytes_)
    exact, mag = f8_lib.exact(clean[1].astype(np.uint8), scales, clean[0].astype(np.float32))
    assert (np.abs(got - exact)[~nan] <= f8_lib.bound(k) * mag[~nan]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 20, 140])
def test_scales_of_any_value(gpu, form, rows):
    """Scales of zero, of both signs, of the greatest and least magnitudes; an
    infinite one reaches its own block's columns."""
    k, n = 384, 260
    r = rng(rows)
    bytes_, _ = f8_lib.random_weights(r, n, k)
    x = uniform(r, (rows, k), 1.0)
    scales = np.array([[0.0, 1e-3, -1e-3], [1e-30, 1e-3, -0.0], [1e20, -1e-40, 2.0]], np.float32)
    y = Guarded((rows, n), gpu)
    sdhip.mul_mat_f8(weights(bytes_, gpu), dev(scales, gpu), dev(x, gpu), y.t)
    torch.cuda.synchronize()
    exact, mag = f8_lib.exact(bytes_, scales, x)
    assert (np.abs(y.check() - exact) <= f8_lib.bound(k) * mag).all()
    scales[1, 1] = np.inf
    y = Guarded((rows, n), gpu)
    sdhip.mul_mat_f8(weights(bytes_, gpu), dev(scales, gpu), dev(x, gpu), y.t)
    torch.cuda.synchronize()
    got = y.check()
    assert not np.isfinite(got[:, 128:256]).any() and np.isfinite(got[:, :128]).all() and np.isfinite(got[:, 256:]).all()


def chains(r, gpu, m1, m2, m3, n):
    """Chains of every kind of operand, with their values in float64."""
    bias = uniform(r, (n,), 1.0)
    full = uniform(r, (m3, m2, m1, n), 1.0)
    matrix = uniform(r, (1, m2, 1, n), 1.0)
    row = uniform(r, (m3, m2, m1, 1), 1.0)
    d = [dev(a, gpu) for a in (bias, full, matrix, row)]
    f = [a.astype(np.float64) for a in (bias, full, matrix, row)]

    def silu(v):
        return v / (1.0 + np.exp(-v))

    return [([("add", d[0])], lambda v: v + f[0]),
            ([("add", d[0]), ("silu", None)], lambda v: silu(v + f[0])),
            ([("mul", d[2]), ("add", d[1])], lambda v: v * f[2] + f[1]),
            ([("add", d[3]), ("mul", d[0]), ("add", d[1])], lambda v: (v + f[3]) * f[0] + f[1])]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 1, 1), (3, 2, 2), (50, 1, 3), (70, 2, 2)])
def test_chains(gpu, form, shape):
    m1, m2, m3 = shape
    k, n = 200, 150
    r = rng(m1)
    bytes_, scales = f8_lib.random_weights(r, n, k)
    x = uniform(r, (m3, m2, m1, k), 1.0)
    exact, mag = f8_lib.exact(bytes_, scales, x.reshape(-1, k))
    exact, mag = exact.reshape(m3, m2, m1, n), mag.reshape(m3, m2, m1, n)
    w, s = weights(bytes_, gpu), dev(scales, gpu)
    for steps, of in chains(r, gpu, m1, m2, m3, n):
        for redirected in (False, True):
            y = Guarded((m3, m2, m1, n), gpu)
            out = Guarded((m3, m2, m1, n), gpu)
            if redirected and steps[-1][0] == "silu":
                continue
            sdhip.mul_mat_f8(w, s, dev(x, gpu), y.t, sdhip.epilogue(steps, redirect=out.t if redirected else None))
            torch.cuda.synchronize()
            got = (out if redirected else y).check()
            y.check()
            # Operands are 1 at most; SiLU's slope is below 1.1 and its own error 8 roundings of it.
            assert (np.abs(got - of(exact)) <= 1.1 * (f8_lib.bound(k, 4) * (mag + 3) + 8 * 2.0 ** -24 * (np.abs(exact) + 1))).all()
            if redirected:
                assert np.isnan(y.t.cpu().numpy()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 33, 140])
def test_from_redirect(gpu, form, rows):
    k, n = 300, 140
    r = rng(rows)
    bytes_, scales = f8_lib.random_weights(r, n, k)
    x, res, bias = uniform(r, (rows, k), 1.0), uniform(r, (rows, n), 1.0), uniform(r, (n,), 1.0)
    out, y = dev(res, gpu), unwritten((rows, n), gpu)
    chain = sdhip.epilogue([("add", dev(bias, gpu))], redirect=out, from_redirect=True)
    sdhip.mul_mat_f8(weights(bytes_, gpu), dev(scales, gpu), dev(x, gpu), y, chain)
    torch.cuda.synchronize()
    exact, mag = f8_lib.exact(bytes_, scales, x)
    total = np.abs(res.astype(np.float64)) + np.abs(bias.astype(np.float64))
    assert (np.abs(out.cpu().numpy() - (exact + res.astype(np.float64) + bias)) <= f8_lib.bound(k, 2) * (mag + total)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fuse", [1, 0])
@pytest.mark.parametrize("rows", [1, 2, 16, 17, 60, 129, 300])
def test_gated(gpu, form, rows, fuse):
    """Halves of whole blocks of 128 columns and not, so that a scale's block lies
    across the halves."""
    for k, half in ((128, 128), (200, 1), (640, 70), (100, 129), (320, 200)):
        r = rng(rows + half)
        bytes_, scales = f8_lib.random_weights(r, 2 * half, k)
        x, bias = uniform(r, (rows, k), 1.0), uniform(r, (2 * half,), 1.0)
        y, out = unwritten((rows, 2 * half), gpu), Guarded((rows, half), gpu)
        sdhip.set_tuning(f"f8_form={form},fuse={fuse}" if form else f"fuse={fuse}")
        sdhip.mul_mat_f8_gated(weights(bytes_, gpu), dev(scales, gpu), dev(x, gpu), y, out.t,
                               sdhip.epilogue([("add", dev(bias, gpu))]))
        torch.cuda.synchronize()
        exact, mag = f8_lib.exact(bytes_, scales, x)
        p = exact + bias.astype(np.float64)
        err = f8_lib.bound(k, 1) * (mag + np.abs(bias.astype(np.float64)))
        a, g = p[:, :half], p[:, half:]
        # |GELU| <= |g|, its slope below 1.13; its own error 16 roundings of it.
        allowed = err[:, :half] * np.abs(g) + 1.13 * (np.abs(a) + err[:, :half]) * err[:, half:] + 16 * 2.0 ** -24 * np.abs(a * g)
        assert (np.abs(out.check() - a * gelu64(g)) <= allowed).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 40, 200])
def test_captured_and_replayed(gpu, form, rows):
    """A captured product replayed with new x, the program's own work between."""
    k, n = 640, 150
    r = rng(rows)
    bytes_, scales = f8_lib.random_weights(r, n, k)
    w, s = weights(bytes_, gpu), dev(scales, gpu)
    x, y, eager = torch.zeros((rows, k), device=gpu), unwritten((rows, n), gpu), unwritten((rows, n), gpu)
    work = sdhip.mul_mat_f8(w, s, x, y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sdhip.mul_mat_f8(w, s, x, y, work=work)
    for i in range(3):
        x.copy_(dev(uniform(r, (rows, k), 1.0), gpu))
        sdhip.mul_mat_f8(w, s, x, eager)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager)


@pytest.mark.gpu
def test_several_streams_at_once(gpu):
    """Calls at once on several streams, a work buffer each, give what they give alone."""
    r = rng(5)
    jobs = []
    for rows, k, n in ((1, 1280, 700), (40, 640, 500), (300, 640, 640), (200, 200, 130)):
        bytes_, scales = f8_lib.random_weights(r, n, k)
        w, s, x = weights(bytes_, gpu), dev(scales, gpu), dev(uniform(r, (rows, k), 1.0), gpu)
        alone, y = unwritten((rows, n), gpu), unwritten((rows, n), gpu)
        work = sdhip.mul_mat_f8(w, s, x, alone)
        work = torch.empty_like(work) if work is not None else None
        jobs.append((w, s, x, y, alone, work, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(5):
        for w, s, x, y, _, work, stream in jobs:
            with torch.cuda.stream(stream):
                sdhip.mul_mat_f8(w, s, x, y, work=work)
    torch.cuda.synchronize()
    for *_, y, alone, _, _ in jobs:
        assert torch.equal(y, alone)


@pytest.mark.gpu
def test_work_buffer_checked(gpu):
    sdhip.set_tuning("f8_form=3")  # whose x is laid out
    try:
        lib = sdhip.load()
        w, s = weights(np.zeros((64, 256), np.uint8), gpu), torch.ones((1, 2), device=gpu)
        x, y = torch.zeros((100, 256), device=gpu), unwritten((100, 64), gpu)
        d = [sdhip.desc(t) for t in (w, s, x, y)]
        size = lib.sdhip_mul_mat_f8_work_size(*d)
        assert size > 0
        buf = torch.zeros(size + 16, dtype=torch.uint8, device=gpu)
        for ptr, n in ((None, size), (buf.data_ptr(), size - 1), (buf.data_ptr() + 8, size)):
            assert lib.sdhip_mul_mat_f8(*d, None, ptr, n, sdhip.stream_handle()) == sdhip.ERROR
        sdhip.check(lib.sdhip_mul_mat_f8(*d, None, ctypes.c_void_p(buf.data_ptr()), size, sdhip.stream_handle()), "mul_mat_f8")
        torch.cuda.synchronize()
        assert (y == 0).all()
    finally:
        sdhip.set_tuning("")


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("k", [16, 32, 48, 80, 112, 144, 176, 208, 240, 272, 528])
def test_rows_that_end_within_a_block(gpu, form, k, gated):
    """Rows of whole 16 bytes, read as they lie: what follows each, NaN in the gap between
    them or in the next row, is no part of it."""
    m, n, odd = 70, 134, 5
    r = rng(k)
    bytes_, scales = f8_lib.random_weights(r, n, k)
    bytes_[odd] = 127
    x = uniform(r, (m, k), 1.0)
    for row in (k, k + 16):
        y, out = Guarded((m, n), gpu), Guarded((m, n // 2), gpu)
        if gated:
            sdhip.mul_mat_f8_gated(weights(bytes_, gpu, row), dev(scales, gpu), dev(x, gpu), y.t, out.t)
        else:
            sdhip.mul_mat_f8(weights(bytes_, gpu, row), dev(scales, gpu), dev(x, gpu), y.t)
        torch.cuda.synchronize()
        exact, mag = f8_lib.exact(bytes_, scales, x)
        got = (out if gated else y).check()
        err = f8_lib.bound(k) * mag
        if gated:
            a, g = exact[:, :n // 2], exact[:, n // 2:]
            err = err[:, :n // 2] * np.abs(g) + 1.13 * (np.abs(a) + err[:, :n // 2]) * err[:, n // 2:] + 16 * 2.0 ** -24 * np.abs(a * g)
            exact = a * gelu64(g)
        others = np.arange(got.shape[1]) != odd
        assert np.isnan(got[:, odd]).all()
        assert (np.abs(got - exact) <= err)[:, others].all()
