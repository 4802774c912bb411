"""ctypes binding of libsdhip.so (include/sdhip.h) for tests and the bench.

Tensors are described as ggml describes them: ne[] extents with ne[0] the
innermost, nb[] byte strides, and a device pointer.  `desc(t)` makes that
descriptor from a torch tensor (ne reversed from torch's shape, strides in
bytes).  Every call goes to the HIP library; nothing here computes.
"""

import ctypes
import os

import torch

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libsdhip.so")

TYPE_F32 = 0
TYPE_F16 = 1
TYPE_Q4_0 = 2
TYPE_Q4_1 = 3
BLOCK = 32  # weights of a block of Q4_0 or Q4_1 ...
BLOCK_BYTES = {TYPE_Q4_0: 18, TYPE_Q4_1: 20}  # ... and its bytes
OK, UNSUPPORTED, ERROR = 0, 1, 2
STEP_ADD, STEP_MUL, STEP_SILU = 0, 1, 2
MAX_STEPS = 6
ROW_NORM_NONE, ROW_NORM_LAYER, ROW_NORM_RMS = 0, 1, 2


class Tensor(ctypes.Structure):
    _fields_ = [
        ("type", ctypes.c_int32),
        ("ne", ctypes.c_int64 * 4),
        ("nb", ctypes.c_int64 * 4),
        ("data", ctypes.c_void_p),
    ]


class Step(ctypes.Structure):
    _fields_ = [("kind", ctypes.c_int32), ("operand", Tensor)]


class Epilogue(ctypes.Structure):
    _fields_ = [
        ("count", ctypes.c_int32),
        ("steps", Step * MAX_STEPS),
        ("redirect", ctypes.POINTER(Tensor)),
        ("from_redirect", ctypes.c_int32),
    ]


class RowNorm(ctypes.Structure):
    """sdhip_row_norm: a norm of rows and what it is multiplied by and added."""

    _fields_ = [
        ("kind", ctypes.c_int32),
        ("eps", ctypes.c_float),
        ("weight_offset", ctypes.c_float),
        ("weight", ctypes.POINTER(Tensor)),
        ("bias", ctypes.POINTER(Tensor)),
    ]


MAX_SRC = 10
MAX_OP_PARAMS = 16


class Node(ctypes.Structure):
    """sdhip_node: a node of a ggml graph as the planner reads it."""


Node._fields_ = [
    ("op", ctypes.c_int32),
    ("unary", ctypes.c_int32),
    ("flags", ctypes.c_int32),
    ("op_params", ctypes.c_int32 * MAX_OP_PARAMS),
    ("tensor", Tensor),
    ("src", ctypes.POINTER(Node) * MAX_SRC),
    ("view_src", ctypes.POINTER(Node)),
]


class NodePlan(ctypes.Structure):
    _fields_ = [
        ("taken", ctypes.c_int32),
        ("count", ctypes.c_int32),
        ("chain", Epilogue),
        ("gated_out", ctypes.POINTER(Node)),
    ]


_T = ctypes.POINTER(Tensor)
_E = ctypes.POINTER(Epilogue)
_R = ctypes.POINTER(RowNorm)
_P = ctypes.c_void_p
_SZ = ctypes.c_size_t
_I6 = ctypes.c_int32 * 6

# (name, restype, argtypes) of every symbol sdhip.h declares.
SIGNATURES = [
    ("sdhip_init", ctypes.c_int, [ctypes.c_int]),
    ("sdhip_last_error", ctypes.c_char_p, []),
    ("sdhip_set_tuning", ctypes.c_int, [ctypes.c_char_p]),
    ("sdhip_get_tuning", ctypes.c_int, [ctypes.c_char_p]),
    ("sdhip_forget", None, [_P, _SZ]),
    ("sdhip_store_arena", None, [_P, _SZ]),
    ("sdhip_store_used", _SZ, [ctypes.POINTER(_SZ)]),
    ("sdhip_profile_enable", None, [ctypes.c_int]),
    ("sdhip_profile_reset", None, []),
    ("sdhip_profile_collect", ctypes.c_int, []),
    ("sdhip_profile_entry", ctypes.c_int,
     [ctypes.c_int, ctypes.POINTER(ctypes.c_char_p), ctypes.POINTER(ctypes.c_double), ctypes.POINTER(ctypes.c_int64)]),
    ("sdhip_mul_mat_supported", ctypes.c_int, [_T, _T, _T]),
    ("sdhip_mul_mat_work_size", _SZ, [_T, _T, _T]),
    ("sdhip_mul_mat", ctypes.c_int, [_T, _T, _T, _E, _P, _SZ, _P]),
    ("sdhip_mul_mat_gated_supported", ctypes.c_int, [_T, _T, _T, _T]),
    ("sdhip_mul_mat_gated", ctypes.c_int, [_T, _T, _T, _E, _T, _P, _SZ, _P]),
    ("sdhip_conv2d_supported", ctypes.c_int, [_T, _T, _T, _I6]),
    ("sdhip_conv2d_path", ctypes.c_int, [_T, _T, _T, _I6]),
    ("sdhip_conv2d_work_size", _SZ, [_T, _T, _T, _I6]),
    ("sdhip_conv2d", ctypes.c_int, [_T, _T, _T, _I6, _E, _P, _SZ, _P]),
    ("sdhip_attention_supported", ctypes.c_int, [_T, _T, _T, _T, ctypes.c_float, ctypes.c_float]),
    ("sdhip_attention_work_size", _SZ, [_T, _T, _T, _T]),
    ("sdhip_attention", ctypes.c_int,
     [_T, _T, _T, _T, ctypes.c_float, ctypes.c_float, ctypes.c_float, _P, _SZ, _P]),
    ("sdhip_group_norm_supported", ctypes.c_int, [_T, _T, ctypes.c_int]),
    ("sdhip_group_norm_work_size", _SZ, [_T, _T, ctypes.c_int]),
    ("sdhip_group_norm", ctypes.c_int, [_T, _T, ctypes.c_int, ctypes.c_float, _E, _P, _SZ, _P]),
    ("sdhip_group_norm_static", ctypes.c_int, [_T, _T, ctypes.c_int, ctypes.c_float, _E, _P]),
    ("sdhip_norm_supported", ctypes.c_int, [_T, _T]),
    ("sdhip_norm", ctypes.c_int, [_T, _T, ctypes.c_float, _E, _P]),
    ("sdhip_norm_residual_supported", ctypes.c_int, [_T, _R, _T, _T, _T, _R, _T]),
    ("sdhip_norm_residual", ctypes.c_int,
     [_T, _R, _T, ctypes.c_float, _T, ctypes.c_float, _T, _R, _T, _P]),
    ("sdhip_plan_nodes", ctypes.c_int,
     [ctypes.POINTER(ctypes.POINTER(Node)), ctypes.c_int, ctypes.c_int, ctypes.POINTER(NodePlan)]),
    ("sdhip_compute_nodes", ctypes.c_int,
     [ctypes.POINTER(ctypes.POINTER(Node)), ctypes.c_int, ctypes.c_int, _P, _SZ, _P]),
    ("sdhip_node_work_size", ctypes.c_int, [ctypes.POINTER(Node), ctypes.POINTER(_SZ)]),
    ("sdhip_token_downsampling", ctypes.c_int, [ctypes.c_int64, ctypes.c_int64]),
]

_lib = None


def load():
    """The library, loaded once; raises if it was not built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} is missing: build it (make -C stable-diffusion.assembly_amd)")
        lib = ctypes.CDLL(LIB_PATH)
        for name, res, args in SIGNATURES:
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _lib = lib
    return _lib


class SdhipError(RuntimeError):
    def __init__(self, status, what):
        super().__init__(f"{what}: status {status}: {load().sdhip_last_error().decode()}")
        self.status = status


def check(status, what):
    if status != OK:
        raise SdhipError(status, what)


def _block_desc(t):
    """The descriptor of 4-bit weights: bytes [N, K / 32, 18] (Q4_0) or
    [N, K / 32, 20] (Q4_1), each row's blocks side by side."""
    types = {size: code for code, size in BLOCK_BYTES.items()}
    if t.dim() != 3 or t.shape[2] not in types:
        raise ValueError(f"4-bit weights are bytes [N, K / {BLOCK}, 18 or 20], not {list(t.shape)}")
    n, blocks, size = t.shape
    if t.stride(2) != 1 or t.stride(1) != size:
        raise ValueError("the blocks of a row of 4-bit weights are not side by side")
    row = t.stride(0)
    return view_desc(t.data_ptr(), types[size], [BLOCK * blocks, n, 1, 1], [size, row, row * n, row * n])


def desc(t):
    """The ggml descriptor of a torch tensor of at most 4 dimensions; of bytes
    [N, K / 32, 18] or [N, K / 32, 20], that of the N x K weights of 4 bits
    (Q4_0, Q4_1) that they hold."""
    if t.dtype == torch.uint8:
        return _block_desc(t)
    if t.dim() > 4:
        raise ValueError("at most 4 dimensions")
    d = Tensor()
    if t.dtype == torch.float32:
        d.type, size = TYPE_F32, 4
    elif t.dtype == torch.float16:
        d.type, size = TYPE_F16, 2
    else:
        raise ValueError(f"type {t.dtype}")
    shape = list(t.shape)[::-1]
    strides = [s * size for s in list(t.stride())[::-1]]
    for k in range(4):
        if k < len(shape):
            d.ne[k] = shape[k]
            d.nb[k] = strides[k]
        else:
            d.ne[k] = 1
            d.nb[k] = d.nb[k - 1] * d.ne[k - 1] if k > 0 else size
    d.data = t.data_ptr()
    return d


def view_desc(data_ptr, dtype_code, ne, nb):
    d = Tensor()
    d.type = dtype_code
    for k in range(4):
        d.ne[k] = ne[k]
        d.nb[k] = nb[k]
    d.data = data_ptr
    return d


def epilogue(steps=(), redirect=None, from_redirect=False):
    """steps: ('add'|'mul', tensor) or ('silu', None); redirect: a torch tensor."""
    e = Epilogue()
    e.count = len(steps)
    e._held = [operand for _, operand in steps] + [redirect]  # kept alive with the epilogue
    kinds = {"add": STEP_ADD, "mul": STEP_MUL, "silu": STEP_SILU}
    for i, (kind, operand) in enumerate(steps):
        e.steps[i].kind = kinds[kind]
        if operand is not None:
            e.steps[i].operand = desc(operand)
    if redirect is not None:
        e._redirect_desc = desc(redirect)  # kept alive with the epilogue
        e.redirect = ctypes.pointer(e._redirect_desc)
    e.from_redirect = 1 if from_redirect else 0
    return e


def stream_handle():
    """torch's current stream on the current device, as the library takes it:
    by torch's own accessor of the handle, since making a torch.cuda.Stream of it
    took 2.9 us of a call's 6.8, this 0.3."""
    return ctypes.c_void_p(torch._C._cuda_getCurrentRawStream(torch.cuda.current_device()))


def set_tuning(text=""):
    check(load().sdhip_set_tuning(text.encode()), "set_tuning")


def get_tuning(name):
    return load().sdhip_get_tuning(name.encode())


def _work(nbytes, device):
    if nbytes == 0:
        return None, 0
    buf = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return buf, nbytes


def mul_mat(w, x, y, chain=None, work=None):
    """y (ne = [N, M...]) = x W^T with the chain; w: [N, K] f16 or f32, or 4-bit
    weights as bytes (desc); x: [..., K] f32."""
    lib = load()
    dw, dx, dy = desc(w), desc(x), desc(y)
    size = lib.sdhip_mul_mat_work_size(dw, dx, dy)
    buf = work
    if buf is None:
        buf, _ = _work(size, x.device)
    ptr = buf.data_ptr() if buf is not None else None
    check(lib.sdhip_mul_mat(dw, dx, dy, ctypes.byref(chain) if chain else None, ptr, size, stream_handle()),
          "mul_mat")
    return buf


def mul_mat_gated(w, x, y, out, chain=None, work=None):
    lib = load()
    dw, dx, dy, do = desc(w), desc(x), desc(y), desc(out)
    size = lib.sdhip_mul_mat_work_size(dw, dx, dy)
    buf = work
    if buf is None:
        buf, _ = _work(size, x.device)
    ptr = buf.data_ptr() if buf is not None else None
    check(lib.sdhip_mul_mat_gated(dw, dx, dy, ctypes.byref(chain) if chain else None, do, ptr, size,
                                  stream_handle()), "mul_mat_gated")
    return buf


def conv_params(s0=1, s1=1, p0=0, p1=0, d0=1, d1=1):
    return _I6(s0, s1, p0, p1, d0, d1)


def conv2d_path(kernel, x, y, params):
    return load().sdhip_conv2d_path(desc(kernel), desc(x), desc(y), params)


def conv2d(kernel, x, y, params, chain=None, work=None):
    lib = load()
    dk, dx, dy = desc(kernel), desc(x), desc(y)
    size = lib.sdhip_conv2d_work_size(dk, dx, dy, params)
    buf = work
    if buf is None:
        buf, _ = _work(size, x.device)
    ptr = buf.data_ptr() if buf is not None else None
    check(lib.sdhip_conv2d(dk, dx, dy, params, ctypes.byref(chain) if chain else None, ptr, size,
                           stream_handle()), "conv2d")
    return buf


def attention(q, k, v, y, scale, work=None):
    lib = load()
    dq, dk, dv, dy = desc(q), desc(k), desc(v), desc(y)
    size = lib.sdhip_attention_work_size(dq, dk, dv, dy)
    buf = work
    if buf is None:
        buf, _ = _work(size, q.device)
    ptr = buf.data_ptr() if buf is not None else None
    check(lib.sdhip_attention(dq, dk, dv, dy, scale, 0.0, 0.0, ptr, size, stream_handle()), "attention")
    return buf


def group_norm(x, y, groups, eps, chain=None, work=None):
    lib = load()
    dx, dy = desc(x), desc(y)
    size = lib.sdhip_group_norm_work_size(dx, dy, groups)
    buf = work
    if buf is None:
        buf, _ = _work(size, x.device)
    ptr = buf.data_ptr() if buf is not None else None
    check(lib.sdhip_group_norm(dx, dy, groups, eps, ctypes.byref(chain) if chain else None, ptr, size,
                               stream_handle()), "group_norm")
    return buf


def group_norm_static(x, y, groups, eps, chain=None):
    """sdhip_group_norm_static: no work buffer, the library's static scratch."""
    check(load().sdhip_group_norm_static(desc(x), desc(y), groups, eps, ctypes.byref(chain) if chain else None,
                                         stream_handle()), "group_norm_static")


def norm(x, y, eps, chain=None):
    check(load().sdhip_norm(desc(x), desc(y), eps, ctypes.byref(chain) if chain else None, stream_handle()),
          "norm")


def row_norm(kind="none", eps=0.0, weight=None, bias=None, weight_offset=0.0):
    """A norm for norm_residual: 'none', 'layer' or 'rms', times (weight +
    weight_offset), plus bias (torch tensors that broadcast over the rows)."""
    r = RowNorm()
    r.kind = {"none": ROW_NORM_NONE, "layer": ROW_NORM_LAYER, "rms": ROW_NORM_RMS}[kind]
    r.eps = eps
    r.weight_offset = weight_offset
    descs = [desc(t) if t is not None else None for t in (weight, bias)]
    r._held = (descs, weight, bias)  # kept alive with the norm
    for name, d in zip(("weight", "bias"), descs):
        if d is not None:
            setattr(r, name, ctypes.pointer(d))
    return r


def norm_residual(y, residual, sum=None, out=None, post=None, pre=None, gate=None, branch_scale=1.0,
                  residual_scale=1.0):
    """sum = residual_scale residual + branch_scale (gate post(y)), out = pre(sum);
    post and pre from row_norm, y, sum and out tensors or None."""
    dy, ds, do, dg = (desc(t) if t is not None else None for t in (y, sum, out, gate))
    check(load().sdhip_norm_residual(dy, post, dg, branch_scale, desc(residual), residual_scale, ds, pre, do,
                                     stream_handle()), "norm_residual")


def profile_enable(on=True):
    load().sdhip_profile_enable(1 if on else 0)


def profile_reset():
    load().sdhip_profile_reset()


def profile_collect():
    """{kernel name: (total ms, launches)} of the launches since the reset."""
    lib = load()
    count = lib.sdhip_profile_collect()
    out = {}
    for i in range(count):
        name = ctypes.c_char_p()
        ms = ctypes.c_double()
        n = ctypes.c_int64()
        if lib.sdhip_profile_entry(i, ctypes.byref(name), ctypes.byref(ms), ctypes.byref(n)):
            out[name.value.decode()] = (ms.value, n.value)
    return out


def store_arena(buf):
    """Give the library `buf` (a uint8 device tensor, or None) as its store."""
    if buf is None:
        load().sdhip_store_arena(None, 0)
    else:
        load().sdhip_store_arena(ctypes.c_void_p(buf.data_ptr()), buf.numel())


def store_used():
    n = ctypes.c_size_t()
    used = load().sdhip_store_used(ctypes.byref(n))
    return used, n.value


def forget(t):
    """sdhip_forget over the memory of tensor t."""
    load().sdhip_forget(ctypes.c_void_p(t.data_ptr()), t.numel() * t.element_size())
