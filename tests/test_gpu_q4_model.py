"""Models of 4-bit weights, and a transformer block modulated by the timestep,
through the library as a program runs them, against float64."""

import math

import pytest
import torch

import sdhip
import unet_step as u
from test_unet import small_config

KINDS = ["q4_0", "q4_1"]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_unet_step(gpu, kind):
    """A whole step; the timestep embedding's two rows go through the library too."""
    m = u.Model(small_config(), gpu, seed=3, weights=kind)
    x, t, c = m.inputs(seed=4)
    ops = u.HipOps(gpu)
    y = m.forward(ops, x, t, c)
    torch.cuda.synchronize()
    assert not any(w.dtype == torch.uint8 for w in ops.widened.values())
    y64 = m.to_reference("cpu").forward(u.TorchOps(torch.float64), x.cpu().double(), t.cpu(), c.cpu().double())
    err = ((y.cpu().double() - y64).norm() / y64.norm()).item()
    print(f"unet step of {kind} weights: relative L2 error {err:.3g}")
    assert err < 2e-5  # test_gpu_unet.py's bound for the step of FP16 weights


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens", [1, 40, 300])
def test_sdxl_block(gpu, kind, tokens):
    """SDXL's block, captured and replayed, against float64 and its eager run."""
    block = u.SdxlBlock(gpu, channels=256, heads=4, seed=2, weights=kind)
    x = torch.randn((1, tokens, 256), generator=torch.Generator(device=gpu).manual_seed(3), device=gpu)
    ops = u.HipOps(gpu)
    if tokens < 16:
        # One token's attention is its value.
        ops.attention = lambda q, k, v, heads: v.clone()
    graph = u.Graph(lambda: block.forward(ops, x), ops)
    eager = graph.eager().clone()
    for _ in range(2):
        assert torch.equal(graph.run(), eager)
        torch.cuda.synchronize()
    ref = u.SdxlBlock("cpu", channels=256, heads=4, seed=2)
    for name in ("ln1", "ln2", "wq", "wk", "wv", "wo", "ff1", "ff2"):
        v = getattr(block, name)
        setattr(ref, name, tuple(t.cpu() for t in v) if isinstance(v, tuple) else v.cpu())
    y64 = ref.forward(u.TorchOps(torch.float64), x.cpu().double())
    err = ((eager.cpu().double() - y64).norm() / y64.norm()).item()
    print(f"sdxl block of {kind} weights, {tokens} tokens: relative L2 error {err:.3g}")
    assert err <= 1e-5  # test_gpu_unet.py's bound for the block of FP16 weights


def norm64(kind, v, eps):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)


class Modulated:
    """Two blocks of attention and gated feed-forward with a shift, a scale and a
    gate an image from the timestep's embedding, RMS norms after each part, 4-bit
    weights: what runs between the blocks is one norm_residual."""

    def __init__(self, device, kind, c, heads):
        g = torch.Generator(device=device).manual_seed(7)

        def randn(*shape, std=1.0, mean=0.0):
            return mean + std * torch.randn(shape, generator=g, device=device)

        self.c, self.heads = c, heads
        self.emb = (u.quantize(randn(6 * c, c, std=0.02), kind), randn(6 * c, std=0.1))
        self.w = {n: u.quantize(randn(*s, std=0.02), kind)
                  for n, s in (("q", (c, c)), ("k", (c, c)), ("v", (c, c)), ("o", (c, c)), ("f1", (8 * c, c)), ("f2", (c, 4 * c)))}
        self.b1, self.b2 = randn(8 * c, std=0.01), randn(c, std=0.01)
        self.after = [randn(c, std=0.1, mean=1.0) for _ in range(2)]

    def forward(self, ops, x, emb):
        b = x.shape[0]
        m = ops.linear(emb, *self.emb).view(b, 6, self.c)
        shift1, scale1, gate1, shift2, scale2, gate2 = (m[:, i:i + 1].contiguous() for i in range(6))
        n = torch.empty_like(x)
        sdhip.norm_residual(None, x, out=n, pre=sdhip.row_norm("layer", 1e-6, scale1, shift1, 1.0))
        q, k, v = (ops.linear(n, self.w[name]) for name in "qkv")
        y = ops.linear(ops.attention(q, k, v, self.heads), self.w["o"])
        s = torch.empty_like(x)
        sdhip.norm_residual(y, x, s, n, sdhip.row_norm("rms", 1e-6, self.after[0]),
                            sdhip.row_norm("layer", 1e-6, scale2, shift2, 1.0), gate1)
        y = ops.linear(ops.geglu(n, self.w["f1"], self.b1), self.w["f2"], self.b2)
        # The sum in place of what it is added to; no norm after the last.
        sdhip.norm_residual(y, s, s, None, sdhip.row_norm("rms", 1e-6, self.after[1]), None, gate2)
        return s

    def forward64(self, x, emb):
        ops = u.TorchOps(torch.float64)
        x, emb = x.cpu().double(), emb.cpu().double()
        m = ops.linear(emb, *(t.cpu() for t in self.emb)).view(x.shape[0], 6, 1, self.c)
        w = {n: t.cpu() for n, t in self.w.items()}
        n = norm64("layer", x, 1e-6) * (1 + m[:, 1]) + m[:, 0]
        y = ops.linear(ops.attention(*(ops.linear(n, w[name]) for name in "qkv"), self.heads), w["o"])
        s = x + m[:, 2] * norm64("rms", y, 1e-6) * self.after[0].cpu().double()
        n = norm64("layer", s, 1e-6) * (1 + m[:, 4]) + m[:, 3]
        y = ops.linear(ops.geglu(n, w["f1"], self.b1.cpu().double()), w["f2"], self.b2.cpu().double())
        return s + m[:, 5] * norm64("rms", y, 1e-6) * self.after[1].cpu().double()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("batch,tokens,channels", [(2, 77, 256), (1, 300, 320), (3, 17, 128)])
def test_modulated_block(gpu, kind, batch, tokens, channels):
    """The operators as they are used together, captured and replayed with new inputs."""
    model = Modulated(gpu, kind, channels, 4)
    g = torch.Generator(device=gpu).manual_seed(9)
    x = torch.randn((batch, tokens, channels), generator=g, device=gpu)
    emb = torch.randn((batch, channels), generator=g, device=gpu)
    ops = u.HipOps(gpu)
    graph = u.Graph(lambda: model.forward(ops, x, emb), ops)
    for _ in range(3):
        got = graph.run().clone()
        torch.cuda.synchronize()
        assert torch.equal(got, graph.eager())
        want = model.forward64(x, emb)
        err = ((got.cpu().double() - want).norm() / want.norm()).item()
        print(f"modulated block of {kind}, {batch} x {tokens} x {channels}: relative L2 error {err:.3g}")
        # Ten operators one after another, each within 1e-6 of its magnitudes, none of whose norms grows what it is
        # given by more than the weights' sqrt(k) 0.02: 1e-5 of the output.
        assert err <= 1e-5
        x.copy_(torch.randn(x.shape, generator=g, device=gpu))
        emb.copy_(torch.randn(emb.shape, generator=g, device=gpu))
    assert math.isfinite(err)
