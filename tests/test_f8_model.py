"""The models' weights in E4M3 (unet_step.py) on the CPU: they hold what they were
made of to half a step, and a model of them is one of their numbers."""

import numpy as np
import pytest
import torch

import f8_lib
import unet_step as u
from test_unet import small_config


@pytest.mark.parametrize("n,k", [(128, 256), (200, 300), (1, 1), (129, 127)])
def test_scaled_weights_hold_the_weights(n, k):
    w = 0.02 * torch.randn((n, k), generator=torch.Generator().manual_seed(1))
    w[:, k // 2:] = 0 if k > 128 else w[:, k // 2:]
    s = u.scaled(w)
    assert u.extents(s) == (n, k) and s.scales.shape == (-(-n // 128), -(-k // 128))
    wide = u.widen(s, torch.float64)
    assert np.array_equal(wide.numpy(), f8_lib.widen(s.values.view(torch.uint8).numpy(), s.scales.numpy()))
    # Half a step of E4M3, 2^-4 of a number or 2^-10 scales, and the scale's and the division's roundings.
    scale = s.scales.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    assert ((wide - w.double()).abs() <= torch.maximum(w.double().abs() / 16, scale / 1024) * (1 + 2.0 ** -20)).all()


def test_x_is_held_as_the_products_take_it():
    g = torch.Generator().manual_seed(2)
    x = torch.randn((60, 300), generator=g, dtype=torch.float64) * torch.exp2(torch.randint(-130, 100, (60, 1), generator=g).double())
    x[3], x[4, 0], x[5] = 0, 448.0, 448.0 * 2.0 ** 5
    assert np.array_equal(u.held(x).numpy(), f8_lib.held(x.numpy()))
    assert u.held(x[None]).shape == (1, 60, 300)


def test_extents_of_a_model_of_f8():
    """SD1.5's linear layers in E4M3 have the extents of its FP16 ones."""
    half, eighth = (u.Model(u.Config(), "meta", weights=w) for w in ("f16", "f8"))
    for of in (lambda m: m.emb_all[0], lambda m: m.time[0][0], lambda m: m.mid[1]["ff1"][0], lambda m: m.mid[1]["k2"][0]):
        assert of(eighth).dtype == torch.float8_e4m3fn and u.extents(of(eighth)) == tuple(of(half).shape)
    assert eighth.conv_in[0].dtype == torch.float16


def test_model_of_f8_in_torch():
    """A step of it, by the plain nodes, is that of a model of the weights' and of
    x's held numbers."""
    m = u.Model(small_config(), "cpu", seed=3, weights="f8")
    x, t, c = m.inputs(seed=4, dtype=torch.float64)
    y = m.forward(u.TorchOps(torch.float64), x, t, c)

    class Wide(u.TorchOps):
        def linear(self, x, w, bias=None, add=()):
            flat = torch.from_numpy(f8_lib.held(x.reshape(-1, x.shape[-1]).numpy())).reshape(x.shape)
            return super().linear(flat, u.widen(w, torch.float64), bias, add)

    assert torch.equal(y, m.forward(Wide(torch.float64), x, t, c))
    assert {st[n][0].dtype for _, st in m.down[0][0] for n in ("q1", "k2")} == {torch.float8_e4m3fn}
