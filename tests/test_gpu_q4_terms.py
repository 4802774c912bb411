"""What the roundings of MUL_MAT of 4-bit weights are of, in every form: each
number of x is held to 2^-22 of itself or 2^-39 of its row's greatest, and the
sums are of d (q - 8) x and, with Q4_1, of (m + 8 d) x, also where these cancel
to a weight of 0 -- two terms that are together below 2.1 of the greatest
number that the block can hold."""

import numpy as np
import pytest
import torch

import q4_lib
import sdhip
from helpers import dev, rng, uniform, unwritten

FORMS = [(form, 70) for form in range(1, 7)] + [(0, 1), (0, 40), (0, 200)]
K, N = 640, 70


def heads(blocks, d, m):
    """The blocks with these scales and least values."""
    blocks = blocks.copy()
    for i, v in enumerate((d, m)):
        blocks[:, :, 2 * i:2 * i + 2] = v.astype(np.float16)[..., None].view(np.uint8).reshape(*v.shape, 2)
    return blocks


def nibble(blocks, k, q):
    """The blocks with number k of every row's q."""
    blocks = blocks.copy()
    at, j = blocks.shape[2] - 16 + k % 16, k // 32
    old = blocks[:, j, at]
    blocks[:, j, at] = (old & 0xf0) | q if k % 32 < 16 else (old & 0x0f) | (q << 4)
    return blocks


def of_kind(r, signs):
    """Q4_1 blocks whose numbers are all 0 or more: least values of 0, of up to
    ten scales, of 0 with nine numbers in ten 0; and any scales and least values."""
    blocks = q4_lib.random_blocks(r, "q4_1", N, K)
    d = r.uniform(0.001, 0.03, (N, K // 32))
    m = np.zeros_like(d)
    if signs == "above 0":
        m = d * r.uniform(0.0, 10.0, d.shape)
    elif signs == "mostly 0":
        low, high = ((r.random((N, K // 32, 16)) < 0.9).astype(np.uint8) for _ in range(2))
        blocks[:, :, 4:] &= (1 - low) * 15 | (1 - high) * 240
    elif signs == "any":
        d, m = (r.uniform(-0.03, 0.03, d.shape) for _ in range(2))
    return heads(blocks, d, m)


SIGNS = ["from 0", "above 0", "mostly 0", "any"]


@pytest.mark.parametrize("signs", SIGNS)
def test_terms_are_of_a_blocks_greatest(signs):
    """|d (q - 8)| + |m + 8 d| < 2.1 max(|m|, |m + 15 d|): m + 8 d lies between
    the two, and 15 |d| is at most their sum, so 8 |d| at most 16 / 15 of one."""
    blocks = of_kind(rng(1), signs)
    _, parts = q4_lib.widen(blocks)
    d, m = (blocks[:, :, 2 * i:2 * i + 2].copy().view(np.float16).astype(np.float64)[..., 0] for i in range(2))
    greatest = np.maximum(np.abs(m), np.abs(m + 15 * d))
    assert (parts <= 2.1 * np.repeat(greatest, 32, axis=1)).all()


@pytest.mark.parametrize("power", [0, -10, -16, -18, -25, -31])
def test_numbers_of_x_in_two_parts(power):
    """x of 2^power of its row's greatest in two FP16 parts, the greatest in [2^14, 2^15)."""
    s = uniform(rng(2), (100000,), 2.0 ** (14 + power))
    hi = s.astype(np.float16)
    lo = (s - hi.astype(np.float32)).astype(np.float16)
    err = np.abs(s.astype(np.float64) - hi.astype(np.float64) - lo.astype(np.float64))
    assert (err <= np.maximum(2.0 ** -22 * np.abs(s), 2.0 ** -39 * 2.0 ** 14)).all()


def check(gpu, form, rows, blocks, x, what):
    y = unwritten((rows, N), gpu)
    sdhip.set_tuning(f"q4_form={form}")
    try:
        sdhip.mul_mat(dev(blocks, gpu), dev(x, gpu), y)
        torch.cuda.synchronize()
    finally:
        sdhip.set_tuning("")
    exact, mag = q4_lib.exact(blocks, x)
    _, parts = q4_lib.widen(blocks)
    held = 2.0 ** -39 * np.abs(x).astype(np.float64).max(-1)[:, None] * parts.sum(-1)
    err = np.abs(y.cpu().numpy() - exact)
    allowed = q4_lib.bound(K) * mag + held
    w, _ = q4_lib.widen(blocks)
    of_weights = (err / (np.abs(x).astype(np.float64) @ np.abs(w).T + 1e-300)).max()
    print(f"{what}: {(err / allowed).max():.3g} of the bound, {of_weights:.3g} of the weights' own products")
    assert np.isfinite(err).all() and (err <= allowed).all()


@pytest.mark.gpu
@pytest.mark.parametrize("form,rows", FORMS)
@pytest.mark.parametrize("signs", SIGNS)
def test_weights_of_one_sign(gpu, form, rows, signs):
    r = rng(rows + form)
    check(gpu, form, rows, of_kind(r, signs), uniform(r, (rows, K), 1.0), f"form {form}, {rows} rows, {signs}")


@pytest.mark.gpu
@pytest.mark.parametrize("form,rows", FORMS)
@pytest.mark.parametrize("power", [12, 20, 30])
@pytest.mark.parametrize("zero", ["q4_0", "q4_1 of no offset", "q4_1 of two terms"])
def test_weights_of_zero_on_a_great_channel(gpu, form, rows, power, zero):
    """A channel 2^power times as great as the others whose weights are 0: by q =
    8 and no offset, which leaves nothing of it, or by q = 0 and m = 0, two terms of
    8 d that cancel."""
    r = rng(rows + form + power)
    if zero == "q4_0":
        blocks = nibble(q4_lib.random_blocks(r, "q4_0", N, K), 100, 8)
    elif zero == "q4_1 of no offset":
        d = r.uniform(0.001, 0.03, (N, K // 32)).astype(np.float16)
        blocks = nibble(heads(q4_lib.random_blocks(r, "q4_1", N, K), d, -8 * d), 100, 8)
    else:
        blocks = nibble(of_kind(r, "from 0"), 100, 0)
    x = uniform(r, (rows, K), 1.0)
    x[:, 100] = 2.0 ** power
    w, parts = q4_lib.widen(blocks)
    assert (w[:, 100] == 0).all() and ((parts[:, 100] == 0).all() or zero == "q4_1 of two terms")
    check(gpu, form, rows, blocks, x, f"form {form}, {rows} rows, 2^{power}, {zero}")
