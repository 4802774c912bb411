"""Linear layers of fewer than 16 rows, which the reference leaves to ggml: whatever
floating-point type their weights are of, torch computes them; those of 4 bits and of
8-bit floating point the library does."""

import pytest
import torch

import unet_step


def ops():
    """The backend without its device: what is not the library's runs anywhere."""
    o = object.__new__(unet_step.HipOps)
    o.widened = {}
    o.reset()
    return o


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32, torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("rows", [1, 2, 15])
def test_weights_of_any_type(dtype, rows):
    g = torch.Generator().manual_seed(rows)
    w = torch.randn((24, 40), generator=g).to(dtype)
    x, bias = torch.randn((rows, 40), generator=g), torch.randn(24, generator=g)
    add = torch.randn((rows, 24), generator=g)
    y = ops().linear(x, w, bias, add=[add])
    want = x.double() @ w.double().t() + bias.double() + add.double()
    # 40 products and sums and two additions, each off by 2^-24 of what they are of.
    bound = 43 * 2.0 ** -24 * (x.double().abs() @ w.double().abs().t() + bias.double().abs() + add.double().abs())
    assert ((y.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("w", [torch.zeros((32, 2, 18), dtype=torch.uint8), unet_step.scaled(torch.ones(32, 64))])
def test_the_librarys(w, monkeypatch):
    """Asked of the library, from one row up."""
    asked = []

    class Library:
        def __getattr__(self, name):
            asked.append(name)
            return lambda *a: 0

    o = ops()
    o.lib = Library()
    monkeypatch.setattr(unet_step.HipOps, "_work", lambda self, size: (None, 0))
    monkeypatch.setattr(unet_step.sdhip, "stream_handle", lambda: None)
    o.linear(torch.zeros((2, 64)), w)
    assert asked[-1] == ("sdhip_mul_mat" if isinstance(w, torch.Tensor) else "sdhip_mul_mat_f8")
