"""What the products of 4-bit weights and the fused norms take and refuse, on
the CPU: descriptors only, nothing is launched."""

import ctypes

import pytest
import torch

import graph_lib as g
import sdhip

FAKE = 1 << 20
F32, Q4_0, Q4_1 = sdhip.TYPE_F32, sdhip.TYPE_Q4_0, sdhip.TYPE_Q4_1


def rows(*shape, data=FAKE):
    ne = list(reversed(shape)) + [1] * (4 - len(shape))
    nb = [4]
    for k in range(1, 4):
        nb.append(nb[k - 1] * ne[k - 1])
    return sdhip.view_desc(data, F32, ne, nb)


def blocks(kind, n, k, row=None, data=4 * FAKE):
    size = sdhip.BLOCK_BYTES[kind]
    row = k // 32 * size if row is None else row
    return sdhip.view_desc(data, kind, [k, n, 1, 1], [size, row, row * n, row * n])


@pytest.mark.parametrize("kind", [Q4_0, Q4_1])
def test_products_taken(kind):
    lib = sdhip.load()
    for m in (1, 2, 15, 16, 100):
        assert lib.sdhip_mul_mat_supported(blocks(kind, 70, 320), rows(m, 320), rows(m, 70))
        assert lib.sdhip_mul_mat_gated_supported(blocks(kind, 70, 320), rows(m, 320), rows(m, 70, data=64 * FAKE),
                                                 rows(m, 35, data=128 * FAKE))
    assert lib.sdhip_mul_mat_supported(blocks(kind, 1, 32), rows(2, 3, 4, 32), rows(2, 3, 4, 1))
    assert lib.sdhip_mul_mat_supported(blocks(kind, 70, 320, row=1002), rows(1, 320), rows(1, 70))


@pytest.mark.parametrize("kind", [Q4_0, Q4_1])
def test_products_refused(kind):
    lib = sdhip.load()
    size = sdhip.BLOCK_BYTES[kind]
    x, y = rows(4, 320), rows(4, 70)
    good = blocks(kind, 70, 320)
    assert lib.sdhip_mul_mat_supported(good, x, y)
    bad = []
    for change in (("ne", 0, 319), ("ne", 0, 0), ("ne", 1, 0), ("ne", 2, 2), ("ne", 3, 0), ("nb", 0, size + 2),
                   ("nb", 1, 10 * size - 2), ("nb", 1, 10 * size + 1), ("nb", 1, -10 * size)):
        d = blocks(kind, 70, 320)
        getattr(d, change[0])[change[1]] = change[2]
        bad.append(d)
    bad.append(blocks(kind, 70, 320, data=FAKE + 1))
    for d in bad:
        assert not lib.sdhip_mul_mat_supported(d, x, y)
        assert lib.sdhip_mul_mat(d, x, y, None, None, 0, None) == sdhip.UNSUPPORTED
        assert lib.sdhip_mul_mat_work_size(d, x, y) == 0
    assert not lib.sdhip_mul_mat_supported(good, rows(4, 352), y)
    assert not lib.sdhip_mul_mat_supported(good, x, rows(4, 71))
    assert not lib.sdhip_mul_mat_supported(good, x, rows(5, 70))
    assert not lib.sdhip_mul_mat_supported(good, rows(0, 320), rows(0, 70))
    apart = rows(4, 320)
    apart.nb[1] += 4
    assert not lib.sdhip_mul_mat_supported(good, apart, y)
    # N odd, an output of another shape, an output over an operand: not gated.
    assert not lib.sdhip_mul_mat_gated_supported(blocks(kind, 71, 320), x, rows(4, 71), rows(4, 35, data=99 * FAKE))
    assert not lib.sdhip_mul_mat_gated_supported(good, x, y, rows(4, 36, data=99 * FAKE))
    assert not lib.sdhip_mul_mat_gated_supported(good, x, rows(4, 70, data=99 * FAKE), rows(4, 35))


def test_extents_that_a_launch_counts():
    """Up to 2^25 rows of x and of the weights, 2^36 weights, 2^35 outputs."""
    lib = sdhip.load()

    def taken(m, n, k):
        y = 1 << 50
        return bool(lib.sdhip_mul_mat_supported(blocks(Q4_0, n, k), rows(m, k, data=1 << 45), rows(m, n, data=y)))

    most = 1 << 25
    assert taken(most, 1, 32) and not taken(most + 1, 1, 32)
    assert taken(1, most, 32) and not taken(1, most + 1, 32)
    assert taken(1, most, 2048) and not taken(1, most, 2080)
    assert taken(1024, most, 32) and not taken(1025, most, 32)
    assert not taken(1, 1, 1 << 31)
    assert not lib.sdhip_mul_mat_supported(blocks(Q4_0, 1, 32), rows(2, 2, most // 2, 32), rows(2, 2, most // 2, 1))


def test_product_over_an_operand_is_an_error():
    lib = sdhip.load()
    w, x = blocks(Q4_0, 320, 320), rows(4, 320)
    assert lib.sdhip_mul_mat(w, x, x, None, None, 0, None) == sdhip.ERROR
    assert lib.sdhip_mul_mat(w, x, rows(4, 320, data=4 * FAKE + 1000), None, None, 0, None) == sdhip.ERROR
    assert lib.sdhip_mul_mat(w, x, rows(4, 320, data=99 * FAKE + 2), None, None, 0, None) == sdhip.ERROR
    assert lib.sdhip_mul_mat(w, x, rows(4, 320, data=None), None, None, 0, None) == sdhip.ERROR


def test_other_operations_do_not_take_4_bits():
    lib = sdhip.load()
    w = blocks(Q4_0, 320, 320)
    x = rows(4, 320)
    assert not lib.sdhip_mul_mat_supported(rows(70, 320), w, rows(320, 70))
    assert not lib.sdhip_norm_supported(w, w)
    assert not lib.sdhip_group_norm_supported(w, w, 4)
    assert not lib.sdhip_attention_supported(x, w, w, x, 0.0, 0.0)
    assert not lib.sdhip_conv2d_supported(w, x, x, sdhip.conv_params())


def test_descriptors_of_bytes():
    t = torch.zeros((70, 10, 18), dtype=torch.uint8)
    d = sdhip.desc(t)
    assert d.type == Q4_0 and list(d.ne) == [320, 70, 1, 1] and d.nb[0] == 18 and d.nb[1] == 180
    d = sdhip.desc(torch.zeros((70, 16, 20), dtype=torch.uint8)[:, :10])
    assert d.type == Q4_1 and list(d.ne) == [320, 70, 1, 1] and d.nb[0] == 20 and d.nb[1] == 320
    for shape in ((70, 180), (70, 10, 19), (2, 70, 10, 18)):
        with pytest.raises(ValueError):
            sdhip.desc(torch.zeros(shape, dtype=torch.uint8))
    with pytest.raises(ValueError):
        sdhip.desc(torch.zeros((70, 10, 36), dtype=torch.uint8)[:, :, ::2])
    with pytest.raises(ValueError):
        sdhip.desc(torch.zeros((70, 20, 18), dtype=torch.uint8)[:, ::2])


def test_planner_takes_4_bit_products():
    """The planner takes a MUL_MAT node of 4-bit weights from one row up, with its chain."""
    def leaf(d):
        n = sdhip.Node()
        n.op = g.OP["NONE"]
        n.tensor = d
        return n

    w, x, b = leaf(blocks(Q4_0, 64, 320)), leaf(rows(1, 320)), leaf(rows(64, data=32 * FAKE))
    out = rows(1, 64, data=64 * FAKE)
    mul, add = sdhip.Node(), sdhip.Node()
    mul.op, add.op = g.OP["MUL_MAT"], g.OP["ADD"]
    for n in (mul, add):
        n.flags = g.FLAG_COMPUTE
        n.tensor = out
    mul.src[0], mul.src[1] = ctypes.pointer(w), ctypes.pointer(x)
    add.src[0], add.src[1] = ctypes.pointer(mul), ctypes.pointer(b)
    nodes = (ctypes.POINTER(sdhip.Node) * 2)(ctypes.pointer(mul), ctypes.pointer(add))
    plan = sdhip.NodePlan()
    lib = sdhip.load()
    assert lib.sdhip_plan_nodes(nodes, 2, 0, plan) == sdhip.OK
    assert plan.taken == g.OP["MUL_MAT"] and plan.count == 2 and plan.chain.count == 1
    size = ctypes.c_size_t(1 << 40)
    assert lib.sdhip_node_work_size(mul, size) == 1 and size.value < 1 << 40


# ---------------------------------------------------------------- norms


def supported(y=None, residual=None, sum=None, out=None, post=None, pre=None, gate=None):
    return bool(sdhip.load().sdhip_norm_residual_supported(y, post, gate, residual, sum, pre, out))


def norm(kind=sdhip.ROW_NORM_RMS, weight=None, bias=None):
    r = sdhip.RowNorm()
    r.kind, r.eps = kind, 1e-6
    r._held = (weight, bias)
    if weight is not None:
        r.weight = ctypes.pointer(weight)
    if bias is not None:
        r.bias = ctypes.pointer(bias)
    return r


A, B, C, D = (rows(2, 9, 64, data=i * FAKE) for i in (1, 2, 3, 4))


def test_norms_taken():
    assert supported(A, B, C, D, norm(), norm())
    assert supported(A, B, C)
    assert supported(None, B, None, D, pre=norm())
    assert supported(None, B, C, D, pre=norm(sdhip.ROW_NORM_NONE))
    assert supported(A, B, B, A, norm(), norm())
    for operand in (rows(64, data=9 * FAKE), rows(1, data=9 * FAKE), rows(2, 1, 64, data=9 * FAKE),
                    rows(9, 1, data=9 * FAKE), rows(2, 9, 64, data=9 * FAKE)):
        assert supported(A, B, C, D, norm(weight=operand), norm(bias=operand), operand)


def test_norms_refused():
    lib = sdhip.load()
    assert not supported(A, None, C, D, norm(), norm())
    assert not supported(A, B, None, None, norm())
    assert not supported(A, B, C, D, norm())               # out without its norm
    assert not supported(A, B, C, None, norm(), norm())    # a norm without out
    assert not supported(None, B, C, D, norm(), norm())    # a norm of no y
    assert not supported(None, B, C, D, None, norm(), rows(64, data=9 * FAKE))
    for bad in (norm(3), norm(-1), norm(weight=rows(63, data=9 * FAKE)), norm(bias=rows(3, 9, 64, data=9 * FAKE))):
        assert not supported(A, B, C, D, bad, norm())
        assert not supported(A, B, C, D, norm(), bad)
    for shape in ((2, 9, 65), (2, 8, 64), (0, 9, 64), (2, 9, 0)):
        assert not supported(rows(*shape), B, C, D, norm(), norm())
        assert not supported(A, rows(*shape), C, D, norm(), norm())
    half = sdhip.view_desc(FAKE, sdhip.TYPE_F16, [64, 9, 2, 1], [2, 128, 1152, 2304])
    assert not supported(half, B, C, D, norm(), norm())
    assert not supported(A, B, C, D, norm(), norm(weight=sdhip.view_desc(9 * FAKE, sdhip.TYPE_F16, [64, 1, 1, 1],
                                                                         [2, 128, 128, 128])))
    assert not supported(rows(2, 9, 64, data=FAKE + 2), B, C, D, norm(), norm())
    # What is written over what is read, or over itself.
    assert not supported(A, B, rows(2, 9, 64, data=FAKE + 4), D, norm(), norm())
    assert not supported(A, B, C, C, norm(), norm())
    assert not supported(A, B, C, D, norm(weight=rows(64, data=3 * FAKE)), norm())
    assert not supported(A, B, C, D, norm(), norm(), rows(64, data=4 * FAKE + 64))
    tight = rows(2, 9, 64, data=7 * FAKE)
    tight.nb[1] = 4 * 63
    assert not supported(A, B, tight, D, norm(), norm())
    same = rows(2, 9, 64, data=7 * FAKE)
    same.nb[2] = 0
    assert not supported(A, B, same, D, norm(), norm())
    assert supported(same, B, C, D, norm(), norm())        # read: rows may share memory
    none = rows(2, 9, 64, data=None)
    assert lib.sdhip_norm_residual(A, norm(), None, 1.0, none, 1.0, C, norm(), D, None) == sdhip.ERROR
    assert lib.sdhip_norm_residual(A, norm(), None, 1.0, None, 1.0, C, norm(), D, None) == sdhip.UNSUPPORTED


def test_forms_tuning():
    lib = sdhip.load()
    w, x, y = blocks(Q4_0, 320, 320), rows(40, 320), rows(40, 320)
    try:
        for bad in ("q4_form=7", "q4_form=-1"):
            with pytest.raises(sdhip.SdhipError):
                sdhip.set_tuning(bad)
        sizes = []
        for form in range(1, 7):
            sdhip.set_tuning(f"q4_form={form}")
            assert sdhip.get_tuning("q4_form") == form
            sizes.append(lib.sdhip_mul_mat_work_size(w, x, y))
        assert sizes[0] == 0 < sizes[1] < sizes[2] and sizes[2] == sizes[3] == sizes[4] == sizes[5]
    finally:
        sdhip.set_tuning("")
    assert sdhip.get_tuning("q4_form") == 0
    assert lib.sdhip_mul_mat_work_size(w, rows(1, 320), rows(1, 320)) == 0
    big = rows(4000, 320), rows(4000, 320)
    assert lib.sdhip_mul_mat(w, *big[:1], rows(4000, 320, data=99 * FAKE), None, None, 0, None) == sdhip.ERROR
    assert b"work" in lib.sdhip_last_error()
