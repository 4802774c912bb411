"""The norms around a block of rows near single precision's limits, about their
mean and after it, against float64."""

import numpy as np
import pytest
import torch

import sdhip
from helpers import dev, normal, rng, unwritten
from test_gpu_residual import check, run

U = 2.0 ** -24


def rows_of(dim, power):
    v = np.clip(normal(rng(dim), (3, dim)), -3.5, 3.5).astype(np.float64)
    v = (v * 2.0 ** power).astype(np.float32)
    assert np.isfinite(v).all() and (v != 0).mean() > 0.9
    return v


# Each width of a row's kernel, and a row read again for each sum.
DIMS = [4, 96, 700, 1280, 2048, 5001, 8192, 16384, 17000]


@pytest.mark.gpu
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("power", [-140, -130, -101, -99, 98, 102, 126])
def test_after_the_block(gpu, dim, power):
    check(run(gpu, (3, dim), "layer", "rms", eps=0.0, y_np=rows_of(dim, power)), f"layer of 2^{power} {dim}")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("power", [-140, -130, -101, -99, 98, 102, 126])
def test_before_the_block(gpu, kind, dim, power):
    """The norm of the residual alone; scale 1, so that the sum is it, exactly."""
    check(run(gpu, (3, dim), pre=kind, y=False, eps=0.0, scales=(1.0, 1.0), r_np=rows_of(dim, power)),
          f"{kind} of 2^{power} {dim}")


@pytest.mark.gpu
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("place", ["after", "before"])
def test_numbers_further_from_their_mean_than_single_precision_holds(gpu, dim, place):
    """A number of 3e38 in every four, the others -3e38: the mean is -1.5e38, the
    greatest 4.5e38 from it, and the norms sqrt(3) and -1 / sqrt(3)."""
    v = np.full((2, dim), -3e38, np.float32)
    v[:, ::4] = 3e38
    z = v.astype(np.float64)
    z = z - z.mean(-1, keepdims=True)
    z /= np.sqrt((z * z).mean(-1, keepdims=True))
    out = unwritten(v.shape, gpu)
    if place == "after":
        sdhip.norm_residual(dev(v, gpu), torch.zeros(v.shape, device=gpu), out, None, sdhip.row_norm("layer", 0.0))
    else:
        sdhip.norm_residual(None, dev(v, gpu), None, out, pre=sdhip.row_norm("layer", 0.0))
    # The difference (2 roundings), the scale and their product.
    assert (np.abs(out.cpu().numpy() - z) <= 5 * U * np.abs(z)).all()


# Lengths of each width, most of them with 1 / n times the sum of n 1.1's, both rounded, not 1.1.
LENGTHS = [4, 123, 246, 492, 503, 984, 955, 1280, 1910, 1989, 3781, 4096, 4024, 5013, 7562, 15124, 16365, 16384, 19999, 32768]


@pytest.mark.gpu
@pytest.mark.parametrize("dim", LENGTHS)
@pytest.mark.parametrize("power", [-140, -60, 0, 30, 60, 80, 127])
def test_rows_of_one_number(gpu, dim, power):
    """Nothing is left of them about their mean: 0 with an epsilon, however far
    below their magnitude, and 0 / 0 without one."""
    number = np.float32(1.1 * 2.0 ** power)
    v = torch.full((1100 if power == 80 else 2, dim), float(number), device=gpu)
    for eps in (1e-6, 0.0):
        out = torch.full_like(v, 7.0)
        sdhip.norm_residual(None, v, None, out, pre=sdhip.row_norm("layer", eps))
        assert (out == 0).all() if eps else out.isnan().all()
        out = torch.full_like(v, 7.0)
        sdhip.norm_residual(v, torch.zeros_like(v), out, None, sdhip.row_norm("layer", eps))
        assert (out == 0).all() if eps else out.isnan().all()
