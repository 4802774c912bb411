"""Models of E4M3 weights through the library as a program runs them: a UNet step, and
a block of channels-last norms, rotary positions of several axes and attention.

x is rounded to E4M3 in each product, so a run in 64 bits parts from one in 32 wherever
their numbers lie on two sides of a rounding's midpoint.  Each operator is therefore
held against 64 bits of what it was given, and the whole against the block of numbers
not rounded to the roundings' own noise."""

import gc
import math
import weakref

import pytest
import torch

import sdhip
import unet_step as u
from test_unet import small_config


def relative(got, want):
    return ((got.cpu().double() - want).norm() / want.norm()).item()


def host(v):
    if isinstance(v, u.BlockScaled):
        return v.to("cpu")
    if isinstance(v, torch.Tensor):
        return v.cpu().double() if v.dtype == torch.float32 else v.cpu()
    return tuple(host(t) for t in v) if isinstance(v, (tuple, list)) else v


def checked(ops, names, bound):
    """`ops` with each call of `names` held against TorchOps on the same inputs."""
    plain, errors = Plain(), []

    def check(name):
        run = getattr(ops, name)

        def call(*args, **kwargs):
            y = run(*args, **kwargs)
            want = getattr(plain, name)(*(host(a) for a in args), **{k: host(v) for k, v in kwargs.items()})
            errors.append(relative(y, want))
            assert errors[-1] <= bound, f"{name} {tuple(y.shape)}: relative L2 error {errors[-1]:.3g}"
            return y

        setattr(ops, name, call)

    for name in names:
        check(name)
    return ops, errors


def axes_of(d):
    """Three axes of d numbers, a third of the pairs or so each."""
    a = d // 8 * 2
    return (a, a, d - 2 * a), (10000.0, 10000.0, 100.0)


class Block(u.HipOps):
    """The nodes of the block below, by the library."""

    def norm_last(self, x, groups, gamma, beta, silu):
        y = torch.empty_like(x)
        chain = sdhip.epilogue([("mul", gamma), ("add", beta)] + ([("silu", None)] if silu else []))
        dx, dy = sdhip._images(x), sdhip._images(y)
        ptr, size = self._work(self.lib.sdhip_group_norm_last_work_size(dx, dy, groups))
        sdhip.check(self.lib.sdhip_group_norm_last(dx, dy, groups, 1e-6, chain, ptr, size, sdhip.stream_handle()), "group_norm_last")
        return y

    def rms(self, x, weight):
        y = torch.empty_like(x)
        sdhip.norm_residual(None, x, out=y, pre=sdhip.row_norm("rms", 1e-6, weight))
        return y

    def turned(self, x, weight, positions):
        d = x.shape[-1]
        y = torch.empty_like(x)
        dims, bases = axes_of(d)
        sdhip.rope(x.transpose(1, 2), positions, sdhip.rope_axes(dims, bases), y.transpose(1, 2),
                   sdhip.row_norm("rms", 1e-6, weight))
        return y


class Plain(u.TorchOps):
    """The same in 64 bits."""

    def norm_last(self, x, groups, gamma, beta, silu):
        y = self.group_norm(x.movedim(-1, 1), groups, 1e-6, gamma, beta, silu)
        return y.movedim(1, -1)

    def rms(self, x, weight):
        return x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight

    def turned(self, x, weight, positions):
        v, at = self.rms(x, weight), 0
        out = v.clone()
        dims, bases = axes_of(x.shape[-1])
        for axis, (n, base) in enumerate(zip(dims, bases)):
            angle = positions[:, axis, None].double() * base ** (-torch.arange(0, n, 2, dtype=torch.float64) / n)
            c, s = (f(angle)[:, None] for f in (torch.cos, torch.sin))
            a, b = v[..., at:at + n:2], v[..., at + 1:at + n:2]
            out[..., at:at + n:2], out[..., at + 1:at + n:2] = a * c - b * s, b * c + a * s
            at += n
        return out


class Exact(Plain):
    """With no number of x rounded."""

    def linear(self, x, w, bias=None, add=()):
        return super().linear(x, u.widen(w, torch.float64), bias, add)


class ImageBlock:
    """A norm of channels-last latents, a projection in, a block of attention with normed
    and turned queries and keys and a gated feed-forward, and the projection back onto
    the latents."""

    def __init__(self, device, c, heads):
        m = object.__new__(u.Model)
        m.device = m.gdev = device
        m.weights = "f8"
        m.gen = torch.Generator(device=device).manual_seed(5)
        self.c, self.heads = c, heads
        self.norm, self.n1, self.n2 = m._norm(c), m._norm(c)[0], m._norm(c)[0]
        self.nq, self.nk = m._norm(c // heads)[0], m._norm(c // heads)[0]
        self.w_in, self.w_out, self.o, self.f1, self.f2 = m._lin(c, c), m._lin(c, c), m._lin(c, c), m._lin(8 * c, c), m._lin(c, 4 * c)
        self.qkv = [m._linear_w(c, c) for _ in range(3)]

    def forward(self, ops, x, positions):
        b, hh, ww, c = x.shape
        t = ops.linear(ops.norm_last(x, 32, *self.norm, True).reshape(b, hh * ww, c), *self.w_in)
        n = ops.rms(t, self.n1)
        q, k, v = (ops.linear(n, w) for w in self.qkv)
        split = (b, hh * ww, self.heads, c // self.heads)
        q, k = (ops.turned(y.reshape(split), w, positions).reshape(b, hh * ww, c) for y, w in ((q, self.nq), (k, self.nk)))
        t = ops.linear(ops.attention(q, k, v, self.heads), *self.o, add=(t,))
        t = ops.linear(ops.geglu(ops.rms(t, self.n2), *self.f1), *self.f2, add=(t,))
        return ops.linear(t, *self.w_out, add=(x.reshape(t.shape),)).reshape(x.shape)


@pytest.mark.gpu
@pytest.mark.parametrize("batch,h,w,c,heads", [(1, 8, 8, 256, 4), (2, 13, 9, 320, 5), (3, 24, 20, 128, 2)])
def test_image_block(gpu, batch, h, w, c, heads):
    """The operators as they are used together: each against 64 bits, then captured and
    replayed with new inputs."""
    block = ImageBlock(gpu, c, heads)
    g = torch.Generator(device=gpu).manual_seed(9)
    x = torch.randn((batch, h, w, c), generator=g, device=gpu)
    at = torch.stack(torch.meshgrid(torch.arange(1), torch.arange(h), torch.arange(w), indexing="ij"), -1)
    positions = at.reshape(h * w, 3).float().to(gpu)
    # Each operator within 1e-6 of its magnitudes, which are at most the weights' 0.02 sqrt(k) < 1.5 times its
    # output's norm on these numbers of mean zero: 1e-5 has room.
    ops, errors = checked(Block(gpu), ["norm_last", "linear", "geglu", "rms", "turned", "attention"], 1e-5)
    first = block.forward(ops, x, positions)
    assert len(errors) == 14
    ops = Block(gpu)
    graph = u.Graph(lambda: block.forward(ops, x, positions), ops)
    assert torch.equal(graph.run(), first)
    exact = object.__new__(ImageBlock)
    exact.__dict__ = {k: host(v) for k, v in block.__dict__.items()}
    for _ in range(3):
        got = graph.run().clone()
        torch.cuda.synchronize()
        assert torch.equal(got, graph.eager())
        want = exact.forward(Exact(), x.cpu().double(), positions.cpu())
        # A rounding to E4M3 moves a number by 2^-4 of it at most, 0.027 in the mean of squares; the parts that
        # are added to x pass at most seven products one after another, and are no larger than x.
        err = relative(got, want)
        print(f"image block, {batch} x {h} x {w} x {c}: relative L2 distance to numbers not rounded {err:.3g}")
        assert err <= 0.027 * 7
        x.copy_(torch.randn(x.shape, generator=g, device=gpu))


@pytest.mark.gpu
def test_unet_step(gpu):
    """A whole step; the timestep embedding's two rows go through the products too."""
    m = u.Model(small_config(), gpu, seed=3, weights="f8")
    x, t, c = m.inputs(seed=4)
    ops, errors = checked(u.HipOps(gpu), ["linear", "geglu"], 1e-5)
    y = m.forward(ops, x, t, c)
    torch.cuda.synchronize()
    assert not ops.widened and len(errors) > 20
    step = u.Step(m, u.HipOps(gpu), (x, t, c))
    for _ in range(2):
        assert torch.equal(step.run(), y)
        torch.cuda.synchronize()
        assert torch.equal(step.eager(), y)
    assert math.isfinite(y.norm().item())


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 40, 300])
def test_sdxl_block(gpu, tokens):
    """SDXL's block, each product against float64, captured and replayed."""
    block = u.SdxlBlock(gpu, channels=256, heads=4, seed=2, weights="f8")
    x = torch.randn((1, tokens, 256), generator=torch.Generator(device=gpu).manual_seed(3), device=gpu)
    ops, errors = checked(u.HipOps(gpu), ["linear", "geglu"], 1e-5)
    if tokens < 16:
        ops.attention = lambda q, k, v, heads: v.clone()  # one token's attention is its value
    first = block.forward(ops, x)
    assert len(errors) == 6
    plain = u.HipOps(gpu)
    if tokens < 16:
        plain.attention = ops.attention
    graph = u.Graph(lambda: block.forward(plain, x), plain)
    for _ in range(2):
        assert torch.equal(graph.run(), first)
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_graphs_that_are_no_longer_used(gpu):
    """A step's graph goes with its last use, and one in a cycle before another is captured."""
    block = u.SdxlBlock(gpu, channels=128, heads=2, seed=2, weights="f8")
    x = torch.randn((1, 20, 128), device=gpu)

    def graph():
        ops = u.HipOps(gpu)
        return u.Graph(lambda: block.forward(ops, x), ops)

    class Forward:
        def forward(self, ops, x, t, ctx):
            return block.forward(ops, x)

    gone = weakref.ref(u.Step(Forward(), u.HipOps(gpu), (x, None, None)))
    assert gone() is None
    first = graph()
    first.itself, gone = first, weakref.ref(first)
    want = first.run().clone()
    torch.cuda.synchronize()
    del first
    threshold = gc.get_threshold()
    gc.set_threshold(1, 1, 1)
    try:
        again = graph()
    finally:
        gc.set_threshold(*threshold)
    assert gone() is None and gc.isenabled()
    assert torch.equal(again.run(), want)
