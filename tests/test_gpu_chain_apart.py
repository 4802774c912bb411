"""The chain apart (fuse = 0) of outputs of more than 2^32 rows, which channels-last
norms of few channels have: each row by its own image's operand."""

import pytest
import torch

import sdhip


@pytest.mark.gpu
@pytest.mark.parametrize("fuse", [0, 1])
def test_more_rows_than_32_bits_count(gpu, fuse):
    """17 GB of zeros, whose norm is 0, plus a number an image, in place."""
    images, width = 3, 1431655766
    assert images * width == 2 ** 32 + 2
    x = torch.zeros((images, 1, width, 1), device=gpu)
    number = torch.tensor([1.0, 2.0, 3.0], device=gpu).view(images, 1, 1, 1)
    sdhip.set_tuning(f"fuse={fuse}")
    try:
        sdhip.group_norm_last(x, x, 1, 1e-5, sdhip.epilogue([("add", number)]))
        torch.cuda.synchronize()
    finally:
        sdhip.set_tuning("")
    for i in range(images):
        flat = x[i].reshape(-1)
        for at in range(0, width, 1 << 28):
            assert bool((flat[at:at + (1 << 28)] == i + 1.0).all()), (i, at)
