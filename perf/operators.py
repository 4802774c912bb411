"""The cases of the products of 4-bit weights (MUL_MAT of Q4_0 and Q4_1, with
and without the gated GELU after them) and of the norms after and before a
block fused with its gate and residual.

`listed()` names the cases, `draw(rng)` gives others of the same ranges,
`prepare(case, seed)` makes what a program holds before the call, `run(state)`
is one pass, `work(case)` the bytes and operations a pass cannot do without,
`exact(case, seed)` its outputs from the definition in 64 bits.  With `own`
false a pass is made of elementary torch operations in single precision; with
it true, of the library's calls, their descriptors, chains and work buffers
made once, as a program with a fixed graph keeps them.

Weights are in ggml's blocks of 32 along K: Q4_0 is a half-precision scale d
and 16 bytes, w = d (q - 8); Q4_1 is d, a half-precision least value m and 16
bytes, w = d q + m; byte j holds number j of the block in its low four bits
and number 16 + j in its high ones.
"""

import ctypes
import math
import os
import sys

import torch

own = False

GELU_K = 2.0 * math.sqrt(2.0 / math.pi)  # GELU by its tanh form: x / (1 + exp(-GELU_K (x + 0.044715 x^3)))


def _product(name, type, rows, inner, outer, bias, residual):
    return dict(name=name, op="product", type=type, rows=rows, inner=inner, outer=outer, bias=bias, residual=residual)


def _gated(name, type, rows, inner, outer):
    return dict(name=name, op="gated", type=type, rows=rows, inner=inner, outer=outer)


def _norms(name, images, tokens, dim, post, pre, modulated):
    return dict(name=name, op="norms", images=images, tokens=tokens, dim=dim, post=post, pre=pre, modulated=modulated)


def listed():
    return [
        # One row through a projection of SDXL's width: the smallest call, of
        # which a token's pass has many.
        _product("q4_0 1 row 1280-1280", "q4_0", 1, 1280, 1280, True, False),
        # The two rows of the timestep embedding through the ResBlocks'
        # projections of it side by side, as SD1.5's step computes them.
        _product("q4_0 2 rows 1280-20160", "q4_0", 2, 1280, 20160, True, False),
        # One token through the wide layer of a text encoder's feed-forward:
        # bound by its 42 MB of weights.
        _product("q4_1 1 row 4096-16384", "q4_1", 1, 4096, 16384, False, False),
        # A few rows, an odd number of blocks of K and a ragged N.
        _product("q4_1 33 rows 2080-1111", "q4_1", 33, 2080, 1111, True, False),
        # The keys (or values) of cross-attention: the prompt's 77 tokens, twice.
        _product("q4_0 154 rows 768-1280", "q4_0", 154, 768, 1280, False, False),
        # The output projection of SDXL's block with its bias and residual.
        _product("q4_0 1976 rows 1280-1280", "q4_0", 1976, 1280, 1280, True, True),
        # The feed-forward's way back, with bias and residual.
        _product("q4_1 1976 rows 5120-1280", "q4_1", 1976, 5120, 1280, True, True),
        # A text encoder's gated feed-forward for one token.
        _gated("q4_0 gated 1 row 2048-5120", "q4_0", 1, 2048, 10240),
        # SDXL's gated feed-forward: the largest product.
        _gated("q4_0 gated 1976 rows 1280-5120", "q4_0", 1976, 1280, 10240),
        # One token of a text encoder with norms on both sides of each block.
        _norms("norms 1 row 4096", 1, 1, 4096, "rms", "rms", False),
        # A transformer block whose shift, scale and gate come from the
        # timestep, one set an image, at SDXL's sizes.
        _norms("norms modulated 2x988 1280", 2, 988, 1280, "none", "layer", True),
        # A 512x512 image's tokens in a wide model: the largest.
        _norms("norms 2x4096 5120", 2, 4096, 5120, "rms", "rms", False),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["product", "product", "product", "gated", "norms", "norms"])
    if op == "norms":
        while True:
            images, tokens, dim = rng.randint(1, 4), _log_int(rng, 1, 4096), _log_int(rng, 64, 5120)
            if images * tokens * dim <= 2 * 4096 * 5120:
                break
        return dict(op=op, images=images, tokens=tokens, dim=dim, post=rng.choice(["none", "layer", "rms"]),
                    pre=rng.choice(["layer", "rms"]), modulated=rng.random() < 0.5)
    while True:
        rows, inner = _log_int(rng, 1, 8192), 32 * _log_int(rng, 2, 160)
        outer = 2 * _log_int(rng, 32, 10240) if op == "gated" else _log_int(rng, 32, 20480)
        if rows * inner * outer <= 1976 * 1280 * 10240 and rows * (inner + outer) <= 1976 * (1280 + 10240):
            break
    case = dict(op=op, type=rng.choice(["q4_0", "q4_1"]), rows=rows, inner=inner, outer=outer)
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
        return mean + std * torch.randn(shape, generator=self.gen, device=self.device)

    def activations(self, *shape):
        """~N(0, 1), one channel in 64 or so eight times as great, as the
        inputs of a transformer's linear layers have them."""
        x = self.values(*shape)
        great = torch.rand(shape[-1], generator=self.gen, device=self.device) < 1.0 / 64.0
        return torch.where(great, 8.0 * x, x)

    def blocks(self, type, n, k):
        """Weights ~N(0, 0.02) in blocks of 4 bits: bytes [n, k / 32, 18] (Q4_0) or [n, k / 32, 20] (Q4_1)."""
        w = self.values(n, k // 32, 32, std=0.02)
        if type == "q4_0":
            far = w.abs().argmax(dim=-1, keepdim=True)
            heads = [torch.gather(w, -1, far) / -8.0]
            low = -8.0 * heads[0].half().float()
        else:
            least = w.amin(dim=-1, keepdim=True)
            heads = [(w.amax(dim=-1, keepdim=True) - least) / 15.0, least]
            low = least.half().float()
        d = heads[0].half().float()
        q = torch.where(d == 0, torch.zeros_like(w), ((w - low) / d).round()).clamp(0, 15).to(torch.uint8)
        nibbles = q[..., :16] | (q[..., 16:] << 4)
        return torch.cat([h.half().contiguous().view(torch.uint8) for h in heads] + [nibbles], dim=-1).contiguous()


def _inputs(case, seed):
    """The case's tensors by name."""
    src = _Source(seed)
    if case["op"] != "norms":
        rows, k, n = case["rows"], case["inner"], case["outer"]
        t = dict(w=src.blocks(case["type"], n, k), x=src.activations(rows, k))
        if case["op"] == "gated" or case["bias"]:
            t["bias"] = src.values(n, std=0.01)
        if case["op"] == "product" and case["residual"]:
            t["residual"] = src.values(rows, n)
        return t
    b, l, d = case["images"], case["tokens"], case["dim"]
    t = dict(y=src.activations(b, l, d), residual=src.values(b, l, d, std=2.0))
    if case["modulated"]:
        # An image's gate, scale and shift; the scale is of 1 + what is given.
        t.update(gate=src.values(b, 1, d, std=0.5), pre_weight=src.values(b, 1, d, std=0.2),
                 pre_bias=src.values(b, 1, d, std=0.2))
    else:
        t["pre_weight"] = src.values(d, mean=1.0, std=0.1)
    if case["post"] != "none":
        t["post_weight"] = src.values(d, mean=1.0, std=0.1)
    return t


def _eps(case):
    return 1e-6


def _offset(case):
    return 1.0 if case["modulated"] else 0.0


def _scales(case):
    """The branch's and the residual's scales."""
    return (1.0, 1.0) if case["modulated"] else (0.5, 1.25)


# ---------------------------------------------------------------- the passes


def _plain_weights(type, w):
    """[n, k] in single precision."""
    d = w[..., 0:2].contiguous().view(torch.float16).float()
    nibbles = w[..., 2 if type == "q4_0" else 4:]
    q = torch.cat([nibbles & 15, nibbles >> 4], dim=-1).float()
    if type == "q4_0":
        v = (q - 8.0) * d
    else:
        v = q * d + w[..., 2:4].contiguous().view(torch.float16).float()
    return v.reshape(w.shape[0], -1)


def _plain_product(case, t):
    y = t["x"] @ _plain_weights(case["type"], t["w"]).t()
    if "bias" in t:
        y = y + t["bias"]
    if "residual" in t:
        y = y + t["residual"]
    if case["op"] == "gated":
        a, g = y[:, :case["outer"] // 2], y[:, case["outer"] // 2:]
        y = a * (g / (1.0 + torch.exp(-GELU_K * (g + 0.044715 * g * g * g))))
    return y


def _plain_norm(kind, x, eps):
    if kind == "none":
        return x
    if kind == "layer":
        x = x - x.mean(dim=-1, keepdim=True)
    return x / torch.sqrt((x * x).mean(dim=-1, keepdim=True) + eps)


def _plain_norms(case, t):
    branch, kept = _scales(case)
    z = _plain_norm(case["post"], t["y"], _eps(case))
    if "post_weight" in t:
        z = z * t["post_weight"]
    if "gate" in t:
        z = z * t["gate"]
    s = kept * t["residual"] + branch * z
    n = _plain_norm(case["pre"], s, _eps(case)) * (t["pre_weight"] + _offset(case))
    if "pre_bias" in t:
        n = n + t["pre_bias"]
    return s, n


class _Plain:
    def __init__(self, case, t):
        self.case, self.t = case, t

    def run(self):
        return (_plain_norms if self.case["op"] == "norms" else _plain_product)(self.case, self.t)


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
        if case["op"] == "norms":
            self._norms(case, t, sdhip, lib)
        else:
            self._product(case, t, sdhip, lib)

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
        dw, dx, dy = sdhip.desc(t["w"]), sdhip.desc(t["x"]), sdhip.desc(y)
        size = lib.sdhip_mul_mat_work_size(dw, dx, dy)
        work = torch.empty(max(size, 16), dtype=torch.uint8, device=y.device)
        self.held += [y, chain, work]
        buffer = (ctypes.c_void_p(work.data_ptr()), ctypes.c_size_t(size))
        link = ctypes.byref(chain) if steps else None
        if case["op"] == "gated":
            self.out = torch.empty((rows, n // 2), device=y.device)
            self.call = lib.sdhip_mul_mat_gated
            self.args = (dw, dx, dy, link, sdhip.desc(self.out), *buffer)
        else:
            self.out = y if redirect is None else redirect
            self.call = lib.sdhip_mul_mat
            self.args = (dw, dx, dy, link, *buffer)

    def _norms(self, case, t, sdhip, lib):
        branch, kept = _scales(case)
        self.out = (torch.empty_like(t["y"]), torch.empty_like(t["y"]))
        post = sdhip.row_norm(case["post"], _eps(case), weight=t.get("post_weight"))
        pre = sdhip.row_norm(case["pre"], _eps(case), weight=t["pre_weight"], bias=t.get("pre_bias"),
                             weight_offset=_offset(case))
        gate = sdhip.desc(t["gate"]) if "gate" in t else None
        self.call = lib.sdhip_norm_residual
        self.args = (sdhip.desc(t["y"]), post, gate, branch, sdhip.desc(t["residual"]), kept,
                     sdhip.desc(self.out[0]), pre, sdhip.desc(self.out[1]))

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
    if case["op"] == "norms":
        b, l, d = case["images"], case["tokens"], case["dim"]
        operands = (3 * b * d if case["modulated"] else d) + (d if case["post"] != "none" else 0)
        # The two statistics, their products and sums, the scales and the gate.
        return dict(bytes=16 * b * l * d + 4 * operands, flops=16 * b * l * d)
    m, k, n = case["rows"], case["inner"], case["outer"]
    weights = n * (k // 32) * (18 if case["type"] == "q4_0" else 20)
    if case["op"] == "gated":
        return dict(bytes=weights + 4 * (m * k + n + m * n // 2), flops=2 * m * k * n + 8 * m * n)
    return dict(bytes=weights + 4 * (m * k + (n if case["bias"] else 0) + m * n * (2 if case["residual"] else 1)),
                flops=2 * m * k * n + m * n * (case["bias"] + case["residual"]))


# ---------------------------------------------------------------- 64 bits


def _exact_weights(type, w):
    """Number by number: bytes to whole numbers, each half of each byte in its place."""
    n, blocks, size = w.shape
    v = torch.empty((n, blocks, 32), dtype=torch.float64, device=w.device)
    whole = w.to(torch.int32)
    for j in range(16):
        byte = whole[:, :, size - 16 + j]
        v[:, :, j] = (byte % 16).double()
        v[:, :, 16 + j] = torch.div(byte, 16, rounding_mode="floor").double()
    heads = w[:, :, :size - 16].contiguous().view(torch.float16).double()
    v = heads[:, :, :1] * (v - 8.0) if type == "q4_0" else heads[:, :, :1] * v + heads[:, :, 1:2]
    return v.view(n, 32 * blocks)


def _exact_norm(kind, x, eps, weight, bias, offset):
    if kind == "layer":
        var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
        x = (x - mean) * torch.rsqrt(var + eps)
    elif kind == "rms":
        x = x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + eps)
    if weight is not None:
        x = x * (weight.double() + offset)
    return x if bias is None else x + bias.double()


def exact(case, seed):
    t = _inputs(case, seed)
    if case["op"] == "norms":
        branch, kept = _scales(case)
        z = _exact_norm(case["post"], t["y"].double(), _eps(case), t.get("post_weight"), None, 0.0)
        if "gate" in t:
            z = z * t["gate"].double()
        s = t["residual"].double() * kept + z * branch
        return s, _exact_norm(case["pre"], s, _eps(case), t["pre_weight"], t.get("pre_bias"), _offset(case))
    y = t["x"].double() @ _exact_weights(case["type"], t["w"]).t()
    for name in ("bias", "residual"):
        if name in t:
            y = y + t[name].double()
    if case["op"] == "gated":
        a, g = y.chunk(2, dim=-1)
        y = a * 0.5 * g * (1.0 + torch.tanh(0.5 * GELU_K * (g + 0.044715 * g ** 3)))
    return y
