"""The models' 4-bit weights (unet_step.py) on the CPU: the blocks hold what
they were made of to half a step, and a model of them counts as one of FP16."""

import pytest
import torch

import q4_lib
import unet_step as u
from test_unet import small_config


@pytest.mark.parametrize("kind", ["q4_0", "q4_1"])
def test_blocks_hold_the_weights(kind):
    w = 0.02 * torch.randn((50, 320), generator=torch.Generator().manual_seed(1))
    w[3] = 0
    blocks = u.quantize(w, kind)
    assert u.extents(blocks) == (50, 320)
    wide = u.widen(blocks, torch.float64)
    assert torch.equal(wide, torch.from_numpy(q4_lib.widen(blocks.numpy())[0]))
    assert (wide[3] == 0).all()
    # Half a step of d (a whole one at Q4_0's far end, whose 8 is clamped to 7), and what rounding d and the least
    # value to FP16 moves: 2^-11 of 15 steps and of the least.
    d = blocks[..., 0:2].contiguous().view(torch.float16).double().abs().repeat_interleave(32, dim=1).reshape(50, 320)
    err = (wide - w.double()).abs()
    step = 1.0 if kind == "q4_0" else 0.5
    assert (err <= step * d * 1.02 + 2.0 ** -10 * 0.1).all()


def test_extents_of_a_model_of_blocks():
    """SD1.5's linear layers in blocks have the extents of its FP16 ones."""
    half, quarter = (u.Model(u.Config(), "meta", weights=w) for w in ("f16", "q4_0"))
    for of in (lambda m: m.emb_all[0], lambda m: m.time[0][0], lambda m: m.mid[1]["ff1"][0], lambda m: m.mid[1]["k2"][0]):
        assert of(quarter).dtype == torch.uint8 and u.extents(of(quarter)) == tuple(of(half).shape)
    assert quarter.conv_in[0].dtype == torch.float16


@pytest.mark.parametrize("kind", ["q4_0", "q4_1"])
def test_model_of_blocks_in_torch(kind):
    """A step of it, by the plain nodes, is that of a model of the blocks' numbers."""
    m = u.Model(small_config(), "cpu", seed=3, weights=kind)
    x, t, c = m.inputs(seed=4, dtype=torch.float64)
    y = m.forward(u.TorchOps(torch.float64), x, t, c)

    class Wide(u.TorchOps):
        def linear(self, x, w, bias=None, add=()):
            return super().linear(x, u.widen(w, torch.float64), bias, add)

    assert torch.equal(y, m.forward(Wide(torch.float64), x, t, c))
    # Its 48 context channels are no whole blocks: those weights stay FP16.
    kinds = {w.dtype for _, st in m.down[0][0] for name in ("q1", "k2") for w in [st[name][0]]}
    assert kinds == {torch.uint8, torch.float16}
