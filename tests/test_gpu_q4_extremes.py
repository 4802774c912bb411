"""MUL_MAT of 4-bit weights whose x lies near single precision's limits, in
every form, against float64: where the exact outputs are finite, the kernels'
are, within q4_lib.bound."""

import numpy as np
import pytest
import torch

import oracle_lib as orc
import q4_lib
import sdhip
from helpers import dev, rng, uniform, unwritten
from test_gpu_q4 import gelu64

KINDS = ["q4_0", "q4_1"]
# Rows that every form takes (asked for), and by the choice of the size (0).
FORMS = [(form, 70) for form in range(1, 7)] + [(0, 1), (0, 40), (0, 200)]
POWERS = [-140, -130, 120, 125, 126, 127]
K, N = 1056, 70


def operands(kind, rows, power, seed):
    """Rows uniform in +-2^power, with a block of 1.5 2^(power - 1) throughout.
    The weights are so small for great rows, and so great for small ones, that
    every sum is a normal number: 1056 products of 0.5 2^127 and parts of 2^-14
    at most stay below 2^123, and 2^-140 of weights of a hundred above 2^-126."""
    r = rng(seed)
    blocks = q4_lib.random_blocks(r, kind, N, K, scale=60.0 if power < 0 else 2.0 ** -18)
    x = r.uniform(-1.0, 1.0, (rows, K)) * 2.0 ** power
    x[:, 64:96] = 0.75 * 2.0 ** power
    x = x.astype(np.float32)
    assert np.isfinite(x).all()
    return blocks, x


def tuned(form, call):
    sdhip.set_tuning(f"q4_form={form}")
    try:
        call()
        torch.cuda.synchronize()
    finally:
        sdhip.set_tuning("")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("form,rows", FORMS)
@pytest.mark.parametrize("power", POWERS)
def test_product(gpu, kind, form, rows, power):
    blocks, x = operands(kind, rows, power, rows + power + 200)
    exact, mag = q4_lib.exact(blocks, x)
    assert mag.min() > 2.0 ** -126 and mag.max() < 2.0 ** 127
    y = unwritten((rows, N), gpu)
    tuned(form, lambda: sdhip.mul_mat(dev(blocks, gpu), dev(x, gpu), y))
    err = orc.metric(y.cpu().numpy(), exact, mag)
    print(f"{kind} form {form} {rows} rows of 2^{power}: {err:.3g} of {q4_lib.bound(K):.3g}")
    assert err <= q4_lib.bound(K)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("form,rows", FORMS)
@pytest.mark.parametrize("power", POWERS)
def test_gated(gpu, kind, form, rows, power):
    """The products brought to order 1 by a step of the chain, a power of two."""
    blocks, x = operands(kind, rows, power, rows + power + 200)
    exact, mag = q4_lib.exact(blocks, x)
    back = np.float32(2.0 ** min(126, -round(np.log2(np.abs(exact).mean()))))
    y, out = unwritten((rows, N), gpu), unwritten((rows, N // 2), gpu)
    steps = sdhip.epilogue([("mul", dev(np.full((1,), back), gpu))])
    tuned(form, lambda: sdhip.mul_mat_gated(dev(blocks, gpu), dev(x, gpu), y, out, steps))
    p, size = exact * float(back), mag * float(back)
    a, g = p[:, :N // 2], p[:, N // 2:]
    # d(a gelu(g)) <= |gelu| da + |a| 1.13 dg; gelu's own exponential and division, and the product, add 2^-20.
    err = q4_lib.bound(K, 1)
    allowed = np.abs(gelu64(g)) * err * size[:, :N // 2] + 1.13 * np.abs(a) * err * size[:, N // 2:]
    allowed = allowed * (1 + 1e-3) + 2.0 ** -20 * np.abs(a) * np.abs(g) + err * err * size[:, :N // 2] * size[:, N // 2:]
    diff = np.abs(out.cpu().numpy() - a * gelu64(g))
    assert np.isfinite(diff).all() and (diff <= allowed + 1e-30).all()
