"""The cases of the products of 8-bit floating-point weights (MUL_MAT of E4M3
with a scale for each block of 128 x 128, with and without the gated GELU after
them), of the rotary positions of several axes with the heads' norm before them,
and of GROUP_NORM of channels-last tensors with its chain.

`listed()` names the cases, `draw(rng)` gives others of the same ranges,
`prepare(case, seed)` makes what a program holds before the call, `run(state)`
is one pass, `work(case)` the bytes and operations a pass cannot do without,
`exact(case, seed)` its outputs from the definition in 64 bits.  With `own`
false a pass is made of elementary torch operations in single precision; with
it true, of the library's calls, their descriptors, chains and work buffers
made once, as a program with a fixed graph keeps them.

A product's x is single precision and is taken in groups of 128 along K: a group
as q 2^e, e the least whole number, -101 at least, with the group's greatest
magnitude at most 448 2^e, and q E4M3, to nearest with ties to even.
"""

import ctypes
import math
import os
import sys

import torch

own = False

GELU_K = 2.0 * math.sqrt(2.0 / math.pi)  # GELU by its tanh form: x / (1 + exp(-GELU_K (x + 0.044715 x^3)))
BLOCK = 128
LEAST_POWER = -101


def _product(name, rows, inner, outer, bias, residual):
    return dict(name=name, op="product", rows=rows, inner=inner, outer=outer, bias=bias, residual=residual)


def _gated(name, rows, inner, outer):
    return dict(name=name, op="gated", rows=rows, inner=inner, outer=outer)


def _rope(name, batch, grid, heads, axes, order, norm, half, start=0, stretch=1.0, base=10000.0):
    return dict(name=name, op="rope", batch=batch, frames=grid[0], height=grid[1], width=grid[2], heads=heads,
                axes=axes, order=order, norm=norm, half=half, start=start, stretch=stretch, base=base)


def _norm(name, images, height, width, channels, groups, silu):
    return dict(name=name, op="group_norm", images=images, height=height, width=width, channels=channels,
                groups=groups, silu=silu)


def listed():
    return [
        # One row through a projection of SDXL's width: the smallest product.
        _product("f8 1 row 1280-1280", 1, 1280, 1280, True, False),
        # A few rows, K of no whole blocks and a ragged N.
        _product("f8 33 rows 2080-1111", 33, 2080, 1111, True, False),
        # The keys (or values) of cross-attention: the prompt's 77 tokens, twice.
        _product("f8 154 rows 768-1280", 154, 768, 1280, False, False),
        # SDXL's feed-forward's way back, with bias and residual.
        _product("f8 1976 rows 5120-1280", 1976, 5120, 1280, True, True),
        # SDXL's gated feed-forward.
        _gated("f8 gated 1976 rows 1280-5120", 1976, 1280, 10240),
        # A 1024x1024 image's tokens in a wide model: the most operations.
        _product("f8 4096 rows 4096-16384", 4096, 4096, 16384, True, False),
        # A text encoder's token far into its context: a launch's latency.
        _rope("rope 1 token 32x128", 1, (1, 1, 1), 32, "128", "halves", "none", False, start=100000, base=1e6),
        # Queries and keys of a 1024x1024 image's tokens, side by side in the
        # projection's output, with their norms.
        _rope("rope image 64x64 48x128 rms", 1, (1, 64, 64), 48, "16,56,56", "adjacent", "rms", False),
        # A video's keys, held in half precision for the attention; positions
        # stretched from those of the training.
        _rope("rope video 21x30x52 12x128", 1, (21, 30, 52), 12, "44,42,42", "adjacent", "rms", True, stretch=0.75),
        # The UNet's lowest level: the smallest norm.
        _norm("group norm 2x8x8x1280", 2, 8, 8, 1280, 32, False),
        # Its first level's, groups of 10 channels.
        _norm("group norm 2x64x64x320 silu", 2, 64, 64, 320, 32, True),
        # The VAE decoder's last level at 1024x1024.
        _norm("group norm 1x1024x1024x128 silu", 1, 1024, 1024, 128, 32, True),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _draw_axes(rng, dim):
    """Even numbers of dim's numbers for 1 to 3 axes; of one head in four some are left as they are."""
    count, left = rng.randint(1, 3), dim if rng.random() < 0.75 else 2 * rng.randint(3, dim // 2)
    dims = []
    for i in range(count - 1):
        dims.append(2 * rng.randint(1, left // 2 - (count - 1 - i)))
        left -= dims[-1]
    return ",".join(str(d) for d in dims + [left])


def draw(rng):
    op = rng.choice(["product", "product", "product", "gated", "rope", "rope", "group_norm", "group_norm"])
    if op == "rope":
        while True:
            batch, grid = rng.randint(1, 2), (_log_int(rng, 1, 24), _log_int(rng, 1, 64), _log_int(rng, 1, 64))
            heads, dim = _log_int(rng, 1, 64), rng.choice([32, 40, 64, 72, 80, 96, 128, 128, 160, 256])
            if batch * grid[0] * grid[1] * grid[2] * heads * dim <= 21 * 30 * 52 * 12 * 128:
                break
        return dict(op=op, batch=batch, frames=grid[0], height=grid[1], width=grid[2], heads=heads, dim=dim,
                    axes=_draw_axes(rng, dim), order=rng.choice(["adjacent", "halves"]),
                    norm=rng.choice(["none", "rms", "rms", "layer"]), half=rng.random() < 0.3,
                    start=_log_int(rng, 1, 100000) if rng.random() < 0.3 else 0,
                    stretch=rng.choice([1.0, 1.0, 0.75, 0.5]), base=rng.choice([100.0, 10000.0, 1e6]))
    if op == "group_norm":
        while True:
            images, height, width = rng.randint(1, 4), _log_int(rng, 4, 1024), _log_int(rng, 4, 1024)
            groups = rng.choice([8, 16, 32, 32, 32])
            channels = groups * _log_int(rng, 1, 80)
            if channels <= 2560 and images * height * width * channels <= 1024 * 1024 * 128:
                break
        return dict(op=op, images=images, height=height, width=width, channels=channels, groups=groups,
                    silu=rng.random() < 0.5)
    while True:
        rows, inner = _log_int(rng, 1, 8192), _log_int(rng, 64, 5120)
        if rng.random() < 0.5:
            inner = 64 * max(1, inner // 64)
        outer = 2 * _log_int(rng, 32, 8192) if op == "gated" else _log_int(rng, 32, 16384)
        if rows * inner * outer <= 4096 * 4096 * 16384 // 4:
            break
    case = dict(op=op, rows=rows, inner=inner, outer=outer)
    if op == "product":
        case.update(bias=rng.random() < 0.5, residual=rng.random() < 0.5)
    return case


# ---------------------------------------------------------------- inputs


class _Source:
    """Numbers ~N(mean, std) on the GPU, from a seed alone."""

    def __init__(self, seed):
        self.device = torch.device("cuda", torch.cuda.current_device())
        self.gen = torch.Generator(device=self.device).manual_seed(seed)

    def values(self, *shape, std=1.0, mean=0.0):
        x = torch.randn(shape, generator=self.gen, device=self.device)
        x = x.mul_(std) if std != 1.0 else x
        return x.add_(mean) if mean != 0.0 else x

    def activations(self, *shape):
        """~N(0, 1), one channel in 64 or so eight times as great, as the
        inputs of a transformer's linear layers have them."""
        x = self.values(*shape)
        great = torch.rand(shape[-1], generator=self.gen, device=self.device) < 1.0 / 64.0
        return x.mul_(torch.where(great, 8.0, 1.0))

    def weights(self, n, k):
        """Weights ~N(0, 0.02) as E4M3 [n, k], and the scales [n / 128, k / 128]
        that bring each block's greatest to 448."""
        w = self.values(n, k, std=0.02)
        scales = _blocks(w, BLOCK).abs().amax(dim=(1, 3)) / 448.0
        return (w / _spread(scales, n, k)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), scales


def _blocks(w, rows):
    """[n, k] as [n / rows, rows, k / 128, 128], zeros past its ends."""
    n, k = w.shape
    w = torch.nn.functional.pad(w, (0, -k % BLOCK, 0, -n % rows))
    return w.view(w.shape[0] // rows, rows, w.shape[1] // BLOCK, BLOCK)


def _spread(scales, n, k):
    """A block's scale at each of its weights."""
    return scales.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]


def _axes(case):
    return [int(d) for d in case["axes"].split(",")]


def _dim(case):
    """A head's numbers: the axes' where no more are said."""
    return case.get("dim", sum(_axes(case)))


def _tokens(case):
    return case["frames"] * case["height"] * case["width"]


def _positions(case, device):
    """[tokens, axes]: a token's column, row and frame, by the last axes first,
    the first axis from `start` on."""
    grid = torch.meshgrid(*(torch.arange(case[n], device=device) for n in ("frames", "height", "width")), indexing="ij")
    at = torch.stack([g.reshape(-1) for g in grid], dim=-1).float()[:, 3 - len(_axes(case)):] * case["stretch"]
    at[:, 0] += case["start"]
    return at.contiguous()


def _inputs(case, seed):
    """The case's tensors by name."""
    src = _Source(seed)
    if case["op"] == "rope":
        b, l, h, d = case["batch"], _tokens(case), case["heads"], _dim(case)
        # The projection's output, heads side by side, behind them as many of others.
        wide = src.activations(b, l, h * d + h * d // 2)
        t = dict(wide=wide, x=wide[:, :, :h * d].view(b, l, h, d).permute(0, 2, 1, 3), at=_positions(case, src.device))
        if case["norm"] != "none":
            # A weight for each head, as queries and keys side by side have them.
            t["weight"] = src.values(h, 1, d, mean=1.0, std=0.1)
        if case["norm"] == "layer":
            t["bias"] = src.values(h, 1, d, std=0.1)
        return t
    if case["op"] == "group_norm":
        shape = (case["images"], case["height"], case["width"], case["channels"])
        x = src.values(*shape, std=2.0).add_(src.values(case["channels"], std=0.5))
        return dict(x=x, scale=src.values(case["channels"], mean=1.0, std=0.1), shift=src.values(case["channels"], std=0.1))
    rows, k, n = case["rows"], case["inner"], case["outer"]
    w, scales = src.weights(n, k)
    t = dict(w=w, scales=scales, x=src.activations(rows, k))
    if case["op"] == "gated" or case["bias"]:
        t["bias"] = src.values(n, std=0.01)
    if case["op"] == "product" and case["residual"]:
        t["residual"] = src.values(rows, n)
    return t


def _eps(case):
    return 1e-5 if case["op"] == "group_norm" else 1e-6


# ---------------------------------------------------------------- the passes


def _plain_groups(x):
    """x as the product takes it: groups of 128 held in E4M3."""
    g = _blocks(x, 1)
    m, e = torch.frexp(g.abs().amax(dim=-1, keepdim=True))  # the greatest is m 2^e, 0.5 <= m < 1
    e = (e - 9 + (m > 0.875)).clamp(min=LEAST_POWER)
    q = torch.ldexp(g, -e).to(torch.float8_e4m3fn).float()
    return torch.ldexp(q, e).view(x.shape[0], -1)[:, :x.shape[1]]


def _plain_product(case, t):
    w = t["w"].float() * _spread(t["scales"], case["outer"], case["inner"])
    y = _plain_groups(t["x"]) @ w.t()
    if "bias" in t:
        y = y + t["bias"]
    if "residual" in t:
        y = y + t["residual"]
    if case["op"] == "gated":
        a, g = y[:, :case["outer"] // 2], y[:, case["outer"] // 2:]
        y = a * (g / (1.0 + torch.exp(-GELU_K * (g + 0.044715 * g * g * g))))
    return y


def _angles(case, at):
    """[tokens, pairs], in 64 bits: a pair's axis and frequency."""
    dims = torch.tensor(_axes(case), device=at.device)
    axis = torch.repeat_interleave(torch.arange(len(dims), device=at.device), dims // 2)
    first = torch.cumsum(dims // 2, 0) - dims // 2
    pair = torch.arange(axis.numel(), device=at.device) - first[axis]
    return at.double()[:, axis] * torch.exp(pair.double() * (-2.0 * math.log(case["base"])) / dims[axis])


def _plain_rope(case, t):
    x = t["x"]
    if case["norm"] == "layer":
        x = x - x.mean(dim=-1, keepdim=True)
    if case["norm"] != "none":
        x = x / torch.sqrt((x * x).mean(dim=-1, keepdim=True) + _eps(case)) * t["weight"]
    if "bias" in t:
        x = x + t["bias"]
    angles = _angles(case, t["at"])
    c, s, pairs = torch.cos(angles).float(), torch.sin(angles).float(), angles.shape[1]
    y = x.clone()
    if case["order"] == "adjacent":
        a, b = x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]
        y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2] = a * c - b * s, a * s + b * c
    else:
        a, b = x[..., :pairs], x[..., pairs:2 * pairs]
        y[..., :pairs], y[..., pairs:2 * pairs] = a * c - b * s, a * s + b * c
    y = y.permute(0, 2, 1, 3).contiguous()  # tokens first, as the attention's caller holds them
    return y.half() if case["half"] else y


def _plain_group_norm(case, t):
    n, h, w, c = t["x"].shape
    x = t["x"].view(n, h * w, case["groups"], c // case["groups"])
    x = x - x.mean(dim=(1, 3), keepdim=True)
    x = x / torch.sqrt((x * x).mean(dim=(1, 3), keepdim=True) + _eps(case))
    y = x.view(n, h, w, c) * t["scale"] + t["shift"]
    return y / (1.0 + torch.exp(-y)) if case["silu"] else y


class _Plain:
    def __init__(self, case, t):
        self.case, self.t = case, t

    def run(self):
        form = {"rope": _plain_rope, "group_norm": _plain_group_norm}.get(self.case["op"], _plain_product)
        return form(self.case, self.t)


class _Own:
    """One call of the library, everything it takes made once."""

    def __init__(self, case, t):
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        package = os.path.join(root, "stable-diffusion.assembly_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
        import sdhip

        self.sdhip = sdhip
        lib = sdhip.load()
        sdhip.check(lib.sdhip_init(torch.cuda.current_device()), "init")
        self.held = [t]
        {"rope": self._rope, "group_norm": self._group_norm}.get(case["op"], self._product)(case, t, sdhip, lib)

    def _buffer(self, size, device):
        work = torch.empty(max(size, 16), dtype=torch.uint8, device=device)
        self.held.append(work)
        return ctypes.c_void_p(work.data_ptr()), ctypes.c_size_t(size)

    def _product(self, case, t, sdhip, lib):
        rows, n = case["rows"], case["outer"]
        y = torch.empty((rows, n), device=t["x"].device)
        steps = [("add", t["bias"])] if "bias" in t else []
        redirect = None
        if "residual" in t:
            # The residual's addition ends the chain and goes to a tensor of its own.
            redirect = torch.empty_like(y)
            steps.append(("add", t["residual"]))
        chain = sdhip.epilogue(steps, redirect=redirect)
        self.held += [y, chain]
        operands = [sdhip.desc(v) for v in (t["w"], t["scales"], t["x"], y)]
        buffer = self._buffer(lib.sdhip_mul_mat_f8_work_size(*operands), y.device)
        link = ctypes.byref(chain) if steps else None
        if case["op"] == "gated":
            self.out = torch.empty((rows, n // 2), device=y.device)
            self.call = lib.sdhip_mul_mat_f8_gated
            self.args = (*operands, link, sdhip.desc(self.out), *buffer)
        else:
            self.out = y if redirect is None else redirect
            self.call = lib.sdhip_mul_mat_f8
            self.args = (*operands, link, *buffer)

    def _rope(self, case, t, sdhip, lib):
        b, l, h, d = case["batch"], _tokens(case), case["heads"], _dim(case)
        self.out = torch.empty((b, l, h, d), device=t["x"].device, dtype=torch.float16 if case["half"] else torch.float32)
        norm = None
        if case["norm"] != "none":
            norm = sdhip.row_norm(case["norm"], _eps(case), weight=t["weight"], bias=t.get("bias"))
        axes = sdhip.rope_axes(_axes(case), case["base"], case["order"])
        self.call = lib.sdhip_rope
        self.args = (sdhip.desc(t["x"]), norm, sdhip.desc(t["at"]), axes, sdhip.desc(self.out.permute(0, 2, 1, 3)))

    def _group_norm(self, case, t, sdhip, lib):
        self.out = torch.empty_like(t["x"])
        steps = [("mul", t["scale"]), ("add", t["shift"])] + ([("silu", None)] if case["silu"] else [])
        chain = sdhip.epilogue(steps)
        self.held.append(chain)
        x, y = sdhip.desc(t["x"]), sdhip.desc(self.out)
        buffer = self._buffer(lib.sdhip_group_norm_last_work_size(x, y, case["groups"]), t["x"].device)
        self.call = lib.sdhip_group_norm_last
        self.args = (x, y, case["groups"], _eps(case), ctypes.byref(chain), *buffer)

    def run(self):
        self.sdhip.check(self.call(*self.args, self.sdhip.stream_handle()), self.call.__name__)
        return self.out


def prepare(case, seed):
    t = _inputs(case, seed)
    return _Own(case, t) if own else _Plain(case, t)


def run(state):
    return state.run()


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    if case["op"] == "rope":
        d, rows = _dim(case), case["batch"] * _tokens(case) * case["heads"]
        operands = case["heads"] * d * {"none": 0, "rms": 1, "layer": 2}[case["norm"]] + _tokens(case) * len(_axes(case))
        # The norm's sum, root and products, and six operations a pair.
        return dict(bytes=rows * d * (6 if case["half"] else 8) + 4 * operands,
                    flops=rows * d * (3 + {"none": 0, "rms": 4, "layer": 7}[case["norm"]]))
    if case["op"] == "group_norm":
        n = case["images"] * case["height"] * case["width"] * case["channels"]
        # The two statistics, their product, the scale and the shift, SiLU.
        return dict(bytes=8 * n + 8 * case["channels"], flops=n * (8 + 4 * case["silu"]))
    m, k, n = case["rows"], case["inner"], case["outer"]
    weights = n * k + 4 * (-(-n // BLOCK)) * (-(-k // BLOCK))
    if case["op"] == "gated":
        return dict(bytes=weights + 4 * (m * k + n + m * n // 2), flops=2 * m * k * n + 8 * m * n)
    return dict(bytes=weights + 4 * (m * k + (n if case["bias"] else 0) + m * n * (2 if case["residual"] else 1)),
                flops=2 * m * k * n + m * n * (case["bias"] + case["residual"]))


# ---------------------------------------------------------------- 64 bits


def _exact_e4m3(v):
    """Numbers of at most 448 to the nearest of E4M3: three bits behind the first,
    steps of 2^-9 below 2^-6."""
    first = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))
    # log2's rounding: the first bit is where its power says.
    first = torch.where(torch.exp2(first) > v.abs().clamp(min=2.0 ** -6), first - 1, first)
    first = torch.where(torch.exp2(first + 1) <= v.abs(), first + 1, first)
    step = torch.exp2(first - 3)
    return torch.round(v / step) * step


def _exact_product(case, t):
    m, k, n = case["rows"], case["inner"], case["outer"]
    y = torch.zeros((m, n), dtype=torch.float64, device=t["x"].device)
    for b in range(-(-k // BLOCK)):
        part = slice(b * BLOCK, min(k, b * BLOCK + BLOCK))
        x = t["x"][:, part].double()
        greatest = x.abs().amax(dim=1, keepdim=True)
        # The least power of two that holds it: from below, doubled while it does not.
        power = torch.exp2(torch.floor(torch.log2(greatest.clamp(min=1e-300) / 448.0)) - 1).clamp(min=2.0 ** LEAST_POWER)
        for _ in range(3):
            power = torch.where(greatest > 448.0 * power, 2.0 * power, power)
        scale = t["scales"][:, b].double().repeat_interleave(BLOCK)[:n]
        y += (_exact_e4m3(x / power) * power) @ (t["w"][:, part].double() * scale[:, None]).t()
    for name in ("bias", "residual"):
        if name in t:
            y += t[name].double()
    if case["op"] == "gated":
        a, g = y.chunk(2, dim=-1)
        y = a * 0.5 * g * (1.0 + torch.tanh(0.5 * GELU_K * (g + 0.044715 * g ** 3)))
    return y


def _exact_rope(case, t):
    x = t["x"].double()
    if case["norm"] == "layer":
        var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
        x = (x - mean) * torch.rsqrt(var + _eps(case)) * t["weight"].double() + t["bias"].double()
    elif case["norm"] == "rms":
        x = x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + _eps(case)) * t["weight"].double()
    y, pairs = x.clone(), sum(_axes(case)) // 2
    p = 0
    for axis, dims in enumerate(_axes(case)):
        for j in range(dims // 2):
            # The pair's two numbers as one complex one, turned.
            one, two = (2 * p, 2 * p + 1) if case["order"] == "adjacent" else (p, pairs + p)
            angle = t["at"][:, axis].double() / case["base"] ** (2 * j / dims)
            z = torch.complex(x[..., one], x[..., two]) * torch.polar(torch.ones_like(angle), angle)
            y[..., one], y[..., two] = z.real, z.imag
            p += 1
    return y.permute(0, 2, 1, 3).contiguous()


def _exact_group_norm(case, t):
    per = case["channels"] // case["groups"]
    y = torch.empty(t["x"].shape, dtype=torch.float64, device=t["x"].device)
    for g in range(case["groups"]):
        part = slice(g * per, g * per + per)
        x = t["x"][..., part].double()
        var, mean = torch.var_mean(x, dim=(1, 2, 3), correction=0, keepdim=True)
        y[..., part] = (x - mean) * torch.rsqrt(var + _eps(case)) * t["scale"][part].double() + t["shift"][part].double()
    return y * torch.sigmoid(y) if case["silu"] else y


def exact(case, seed):
    form = {"rope": _exact_rope, "group_norm": _exact_group_norm}.get(case["op"], _exact_product)
    return form(case, _inputs(case, seed))
