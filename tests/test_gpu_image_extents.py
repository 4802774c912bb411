"""The products of E4M3 weights, the rotary positions and GROUP_NORM of channels-last
tensors at extents whose addresses pass 32 bits or whose workgroups pass a launch, and
the output's own memory as a chain's operand: parts of the outputs against 64 bits, none
left unwritten."""

import numpy as np
import pytest
import torch

import f8_lib
import sdhip
from helpers import dev, rng, uniform
from test_gpu_f8 import weights
from test_gpu_rope import allowed, reference


def random_bytes(gpu, n, k, seed):
    """E4M3's bytes [n, k], none NaN's."""
    g = torch.Generator(device=gpu).manual_seed(seed)
    w = torch.randint(0, 127, (n, k), dtype=torch.uint8, device=gpu, generator=g)
    return w.add_(torch.randint(0, 2, (n, 1), dtype=torch.uint8, device=gpu, generator=g) * 128)


def some(r, n, count):
    return np.unique(np.concatenate([[0, 1, n // 2, n - 2, n - 1], r.integers(0, n, count)]).clip(0, n - 1))


def product(gpu, m, k, n, form, row=None):
    """Rows and columns of a product of random numbers against 64 bits."""
    r, g = rng(m + k), torch.Generator(device=gpu).manual_seed(m + n)
    x = torch.rand((m, k), generator=g, device=gpu) * 2 - 1
    w = random_bytes(gpu, n, k, n + k)
    if row is not None:
        buf = torch.full((n, row), 127, dtype=torch.uint8, device=gpu)
        buf[:, :k] = w
        w = buf[:, :k]
    s = torch.rand((-(-n // 128), -(-k // 128)), generator=g, device=gpu) * 1e-4
    y = torch.full((m, n), float("nan"), device=gpu)
    sdhip.set_tuning(f"f8_form={form}")
    try:
        sdhip.mul_mat_f8(w.view(torch.float8_e4m3fn), s, x, y)
        torch.cuda.synchronize()
    finally:
        sdhip.set_tuning("")
    count = 60 if k < 100000 else 3
    rows, columns = some(r, m, count), some(r, n, count)
    at_m, at_n = (torch.from_numpy(v).to(gpu) for v in (rows, columns))
    scales = s[at_n // 128].cpu().numpy().astype(np.float64).repeat(128, 1)[:, :k]
    v, q = f8_lib.TABLE[w[at_n].cpu().numpy()] * scales, f8_lib.held(x[at_m].cpu().numpy())
    got = y[at_m][:, at_n].cpu().numpy()
    assert (np.abs(got - q @ v.T) <= f8_lib.bound(k) * (np.abs(q) @ np.abs(v).T)).all()
    assert all(not y[i:i + (1 << 20)].isnan().any() for i in range(0, m, 1 << 20))


@pytest.mark.gpu
@pytest.mark.parametrize("form", range(7))
def test_many_rows(gpu, form):
    """4.4 GB of outputs and, laid out, 4.3 of x; more rows than workgroups lay out at once."""
    product(gpu, 1 << 25, 20, 33, form)


@pytest.mark.gpu
@pytest.mark.parametrize("form", range(7))
def test_many_weights(gpu, form):
    """5 GB of them, 8.6 laid out."""
    product(gpu, 3, 150, (1 << 25) - 5, form)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,form", [(5, 1 << 23, 0), (40, (1 << 22) + 100, 2), (70, 1 << 22, 3), (70, (1 << 22) - 50, 4), (70, 1 << 22, 5), (70, 1 << 22, 6)])
def test_long_rows(gpu, m, k, form):
    product(gpu, m, k, 7, form)


@pytest.mark.gpu
@pytest.mark.parametrize("form", range(7))
@pytest.mark.parametrize("row", [1 << 24, (1 << 24) + 16])
def test_weights_far_apart(gpu, form, row):
    """Rows of 256 in a tensor of 5 GB, at the tiles' furthest and past it."""
    product(gpu, 60, 256, 300, form, row)


@pytest.mark.gpu
@pytest.mark.parametrize("form", range(7))
@pytest.mark.parametrize("rows", [1, 40, 200])
def test_output_as_operand(gpu, form, rows):
    """y = x W^T + b + y in y's own memory."""
    k, n = 640, 150
    r = rng(rows)
    bytes_, scales = f8_lib.random_weights(r, n, k)
    x, bias, before = uniform(r, (rows, k), 1.0), uniform(r, (n,), 1.0), uniform(r, (rows, n), 1.0)
    y = dev(before, gpu)
    sdhip.set_tuning(f"f8_form={form}")
    try:
        sdhip.mul_mat_f8(weights(bytes_, gpu), dev(scales, gpu), dev(x, gpu), y, sdhip.epilogue([("add", dev(bias, gpu)), ("add", y)]))
        torch.cuda.synchronize()
    finally:
        sdhip.set_tuning("")
    exact, mag = f8_lib.exact(bytes_, scales, x)
    mag = mag + np.abs(bias) + np.abs(before)
    assert (np.abs(y.cpu().numpy() - (exact + bias + before)) <= f8_lib.bound(k, 2) * mag).all()


def turned(gpu, b, h, l, d, dims, half):
    """Tokens of a rotation [b, h, l, d], laid out by tokens, against 64 bits."""
    g, r = torch.Generator(device=gpu).manual_seed(d), rng(l)
    x = (torch.rand((b, l, h, d), generator=g, device=gpu) * 2 - 1).permute(0, 2, 1, 3)
    at = torch.rand((l, len(dims)), generator=g, device=gpu) * 100
    y = torch.full((b, l, h, d), float("nan"), dtype=torch.float16 if half else torch.float32, device=gpu).permute(0, 2, 1, 3)
    sdhip.rope(x, at, sdhip.rope_axes(dims), y, sdhip.row_norm("rms", 1e-6))
    torch.cuda.synchronize()
    tokens, heads = some(r, l, 40), some(r, h, 40)
    t, hd = torch.from_numpy(tokens).to(gpu), torch.from_numpy(heads).to(gpu)
    want, size = reference(x[:, :, t][:, hd].cpu().numpy(), at[t].cpu().numpy()[None], dims, 10000.0, "adjacent", False, "rms", np.float64(np.float32(1e-6)),
                           offset=0.0, weight=None, bias=None)
    got = y[:, :, t][:, hd].cpu().numpy().astype(np.float64)
    assert (np.abs(got - want) <= allowed(want, size, half)).all()
    flat = y.permute(0, 2, 1, 3).reshape(-1)
    assert all(not flat[i:i + (1 << 28)].isnan().any() for i in range(0, flat.numel(), 1 << 28))


@pytest.mark.gpu
@pytest.mark.parametrize("b,h,l,d,dims", [(1, 16, 1 << 21, 64, [16, 24, 24]), (2, 3, 3 << 20, 128, [128]), (1, 1 << 24, 3, 2, [2])])
@pytest.mark.parametrize("half", [False, True])
def test_many_tokens_and_heads(gpu, b, h, l, d, dims, half):
    turned(gpu, b, h, l, d, dims, half)


def normed(gpu, shape, groups, images):
    """Images of a norm against 64 bits, by chunks of its pixels."""
    n, h, w, c = shape
    g = torch.Generator(device=gpu).manual_seed(c)
    x = torch.rand(shape, generator=g, device=gpu) * 2 - 1
    y = torch.full(shape, float("nan"), device=gpu)
    sdhip.group_norm_last(x, y, groups, 1e-5)
    torch.cuda.synchronize()
    per = -(-c // groups)
    for i in images:
        rows, got = x[i].reshape(-1, c), y[i].reshape(-1, c)
        chunks = [slice(p, p + (1 << 22)) for p in range(0, h * w, 1 << 22)]
        # Sums of a group's channels: [groups, per], zeros past the channels.
        total = torch.zeros((2, -(-c // per) * per), dtype=torch.float64, device=gpu)
        for s in chunks:
            v = rows[s].double()
            total[0, :c] += v.sum(0)
            total[1, :c] += (v * v).sum(0)
        count = torch.zeros(total.shape[1], dtype=torch.float64, device=gpu)
        count[:c] = h * w
        sums, count = total.view(2, -1, per).sum(-1), count.view(-1, per).sum(-1)
        mean = sums[0] / count
        scale = 1 / torch.sqrt(sums[1] / count - mean * mean + np.float64(np.float32(1e-5)))
        mean, scale = (v.repeat_interleave(per)[:c] for v in (mean, scale))
        for s in chunks:
            want = (rows[s].double() - mean) * scale
            # test_gpu_norm_last.py's six roundings, the sums' own in 64 bits far below one.
            assert ((got[s].double() - want).abs() <= 6 * 2.0 ** -24 * want.abs() + 2.0 ** -30).all()
    flat = y.reshape(-1)
    assert all(not flat[i:i + (1 << 28)].isnan().any() for i in range(0, flat.numel(), 1 << 28))


@pytest.mark.gpu
@pytest.mark.parametrize("shape,groups", [((1, 1 << 13, 1 << 13, 24), 3), ((3, 1 << 12, 1 << 12, 30), 7), (((1 << 22) + 3, 1, 2, 8), 2),
                                          (((1 << 16) + 1, 40, 40, 12), 3), ((1, 1, 3, 1 << 24), 5), ((2, 3, 1, 1 << 23), 1 << 23)])
def test_many_pixels_images_and_channels(gpu, shape, groups):
    """6 GB of an image; more images than a launch takes; groups of all channels and of one."""
    normed(gpu, shape, groups, sorted({0, shape[0] // 2, shape[0] - 1}))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 4, 4, 64), (1, 90, 60, 96)])
def test_norm_of_its_output_as_operand(gpu, shape):
    """y = norm(y) + y in y's own memory, by one launch and by two."""
    x = uniform(rng(3), shape, 1.0)
    y, apart = dev(x, gpu), torch.empty(shape, device=gpu)
    sdhip.group_norm_last(dev(x, gpu), apart, 32, 1e-5, sdhip.epilogue([("add", dev(x, gpu))]))
    sdhip.group_norm_last(y, y, 32, 1e-5, sdhip.epilogue([("add", y)]))
    torch.cuda.synchronize()
    assert torch.equal(y, apart)
