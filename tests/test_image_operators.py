"""What the products of E4M3 weights, the rotary positions and GROUP_NORM of
channels-last tensors take and refuse, on the CPU: descriptors only, nothing is
launched."""

import ctypes

import pytest
import torch

import sdhip

FAKE = 1 << 20
F32, F16, F8 = sdhip.TYPE_F32, sdhip.TYPE_F16, sdhip.TYPE_F8_E4M3


def rows(*shape, data=FAKE, type=F32):
    size = 2 if type == F16 else 4
    ne = list(reversed(shape)) + [1] * (4 - len(shape))
    nb = [size]
    for k in range(1, 4):
        nb.append(nb[k - 1] * ne[k - 1])
    return sdhip.view_desc(data, type, ne, nb)


def changed(d, field, k, v):
    c = sdhip.view_desc(d.data, d.type, list(d.ne), list(d.nb))
    if field in ("type", "data"):
        setattr(c, field, v)
    else:
        getattr(c, field)[k] = v
    return c


# ---------------------------------------------------------------- products


def weights(n, k, row=None, data=64 * FAKE):
    row = k if row is None else row
    return sdhip.view_desc(data, F8, [k, n, 1, 1], [1, row, row * n, row * n])


def scales(n, k, row=None, data=32 * FAKE):
    b, row = -(-k // 128), -(-k // 128) if row is None else row
    m = -(-n // 128)
    return sdhip.view_desc(data, F32, [b, m, 1, 1], [4, 4 * row, 4 * row * m, 4 * row * m])


def taken(w, s, x, y):
    return bool(sdhip.load().sdhip_mul_mat_f8_supported(w, s, x, y))


@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 1280, 1280), (15, 100, 129), (16, 128, 128), (5000, 2080, 1111)])
def test_products_taken(m, k, n):
    lib = sdhip.load()
    assert taken(weights(n, k), scales(n, k), rows(m, k), rows(m, n))
    assert taken(weights(n, k, k + 3, 64 * FAKE + 1), scales(n, k, -(-k // 128) + 2), rows(m, k), rows(m, n))
    size = lib.sdhip_mul_mat_f8_work_size(weights(n, k), scales(n, k), rows(m, k), rows(m, n))
    assert size == 0 if m <= 16 else size >= m * k
    if n % 2 == 0:
        assert lib.sdhip_mul_mat_f8_gated_supported(weights(n, k), scales(n, k), rows(m, k, data=1 << 40), rows(m, n, data=1 << 41),
                                                    rows(m, n // 2, data=1 << 42))


def test_forms_of_the_products():
    """f8_form takes the forms there are, and the work buffer follows it."""
    lib = sdhip.load()
    d = weights(320, 512), rows(3, 4, data=2 * FAKE), rows(40, 512, data=4 * FAKE), rows(40, 320, data=16 * FAKE)
    try:
        sizes = []
        for form in range(7):
            sdhip.set_tuning(f"f8_form={form}")
            sizes.append(lib.sdhip_mul_mat_f8_work_size(*d))
        # None for the forms of few rows, x's numbers and powers of whole tiles for the others.
        assert sizes[1] == sizes[2] == 0 and len(set(sizes[3:])) == 1 and sizes[3] >= 128 * (512 + 4 * 4)
        for wrong in ("-1", "7", "x"):
            with pytest.raises(Exception):
                sdhip.set_tuning(f"f8_form={wrong}")
    finally:
        sdhip.set_tuning("")


def test_products_of_matrices_taken():
    assert taken(weights(70, 320), scales(70, 320), rows(2, 3, 4, 320), rows(2, 3, 4, 70))


def test_products_refused():
    lib = sdhip.load()
    w, s, x, y = weights(300, 320), scales(300, 320), rows(4, 320), rows(4, 300)
    assert taken(w, s, x, y)
    bad = [(changed(w, f, k, v), s, x, y) for f, k, v in
           (("type", 0, F32), ("type", 0, sdhip.TYPE_Q4_0), ("type", 0, 0), ("ne", 0, 0), ("ne", 0, 321), ("ne", 1, 0), ("ne", 1, 301),
            ("ne", 2, 2), ("ne", 3, 0), ("nb", 0, 2), ("nb", 1, 319), ("nb", 1, -320))]
    bad += [(w, changed(s, f, k, v), x, y) for f, k, v in
            (("type", 0, F16), ("ne", 0, 2), ("ne", 0, 4), ("ne", 1, 2), ("ne", 1, 4), ("ne", 2, 2), ("ne", 3, 0), ("nb", 0, 8),
             ("nb", 1, 8), ("nb", 1, 14), ("nb", 1, -12))]
    bad += [(w, s, changed(x, f, k, v), y) for f, k, v in
            (("type", 0, F16), ("ne", 0, 319), ("ne", 1, 5), ("ne", 1, 0), ("ne", 2, 2), ("nb", 0, 8), ("nb", 1, 1284))]
    bad += [(w, s, x, changed(y, f, k, v)) for f, k, v in
            (("type", 0, F16), ("ne", 0, 299), ("ne", 1, 5), ("ne", 3, 2), ("nb", 0, 8), ("nb", 1, 1204))]
    bad += [(None, s, x, y), (w, None, x, y), (w, s, None, y), (w, s, x, None)]
    for d in bad:
        assert not taken(*d)
        assert lib.sdhip_mul_mat_f8(*d, None, None, 0, None) == sdhip.UNSUPPORTED
        assert lib.sdhip_mul_mat_f8_work_size(*d) == 0
    odd = weights(301, 320), scales(301, 320), x, rows(4, 301)
    assert taken(*odd) and not lib.sdhip_mul_mat_f8_gated_supported(*odd, rows(4, 150, data=1 << 40))
    assert not lib.sdhip_mul_mat_f8_gated_supported(w, s, x, rows(4, 300, data=1 << 41), rows(4, 151, data=1 << 40))
    assert not lib.sdhip_mul_mat_f8_gated_supported(w, s, x, rows(4, 300, data=1 << 41), rows(4, 150))       # over x
    assert not lib.sdhip_mul_mat_f8_gated_supported(w, s, x, rows(4, 300, data=1 << 41), rows(4, 150, data=32 * FAKE))
    assert not lib.sdhip_mul_mat_f8_gated_supported(w, s, x, rows(4, 300, data=1 << 41), None)


def test_products_that_are_errors():
    lib = sdhip.load()
    w, s, x = weights(320, 320), scales(320, 320), rows(4, 320)

    def call(w=w, s=s, x=x, y=rows(4, 320, data=1 << 40)):
        return lib.sdhip_mul_mat_f8(w, s, x, y, None, None, 0, None)

    assert call(y=x) == sdhip.ERROR
    assert call(y=rows(4, 320, data=64 * FAKE + 1000)) == sdhip.ERROR
    assert call(y=rows(4, 320, data=32 * FAKE + 32)) == sdhip.ERROR
    assert call(y=rows(4, 320, data=(1 << 40) + 2)) == sdhip.ERROR
    assert call(x=rows(4, 320, data=FAKE + 1)) == sdhip.ERROR
    assert call(s=scales(320, 320, data=32 * FAKE + 2)) == sdhip.ERROR
    for name in ("w", "s", "x"):
        d = {"w": w, "s": s, "x": x}[name]
        assert call(**{name: changed(d, "data", 0, None)}) == sdhip.ERROR
    assert call(y=rows(4, 320, data=None)) == sdhip.ERROR
    sdhip.set_tuning("f8_form=3")  # whose x is laid out
    try:
        many = rows(4000, 320), rows(4000, 320, data=1 << 40)
        assert lib.sdhip_mul_mat_f8(w, s, *many, None, None, 0, None) == sdhip.ERROR
        assert b"work" in lib.sdhip_last_error()
        size = lib.sdhip_mul_mat_f8_work_size(w, s, *many)
        for ptr, n in ((1 << 44, size - 1), ((1 << 44) + 8, size)):
            assert lib.sdhip_mul_mat_f8(w, s, *many, None, ptr, n, None) == sdhip.ERROR
    finally:
        sdhip.set_tuning("")


def test_chain_operands_over_the_output():
    """Refused but where an element is read at its own place: the output's memory in its
    layout; with the chain apart that is overwritten before it is read."""
    lib = sdhip.load()
    w, s, x, at = weights(320, 320), scales(320, 320), rows(400, 320), 1 << 40
    y, other = rows(400, 320, data=at), rows(400, 320, data=1 << 41)

    def call(operand, redirect=None, from_redirect=0):
        e = sdhip.Epilogue()
        e.count = 1
        e.steps[0].kind, e.steps[0].operand = 0, operand
        e.from_redirect = from_redirect
        if redirect is not None:
            e.redirect = ctypes.pointer(redirect)
        norm = lib.sdhip_group_norm_last(rows(1, 1, 400, 320), rows(1, 1, 400, 320, data=at), 8, 1e-5, e, None, 0, None)
        return lib.sdhip_mul_mat_f8(w, s, x, y, e, None, 0, None), norm

    try:
        for fuse in (1, 0):
            sdhip.set_tuning(f"f8_form=3,fuse={fuse}")
            for operand in (rows(320, data=at), rows(320, data=at + 4 * 320 * 399), rows(400, 320, data=at + 16), rows(400, 320, data=at - 16)):
                assert call(operand) == (sdhip.UNSUPPORTED, sdhip.UNSUPPORTED)
            # What is taken lacks its work buffer.
            assert call(y)[0] == (sdhip.ERROR if fuse else sdhip.UNSUPPORTED)
            assert call(rows(320, data=1 << 42))[0] == sdhip.ERROR and b"work" in lib.sdhip_last_error()
            assert call(other, redirect=other)[0] == sdhip.ERROR
            assert call(rows(400, 320, data=(1 << 41) + 16), redirect=other)[0] == sdhip.UNSUPPORTED
            assert call(y, redirect=other)[0] == (sdhip.ERROR if fuse else sdhip.UNSUPPORTED)
            assert call(rows(320, data=1 << 42), redirect=rows(400, 320))[0] == sdhip.ERROR and b"lies over" in lib.sdhip_last_error()
    finally:
        sdhip.set_tuning("")


def test_extents_that_a_launch_counts():
    """Up to 2^25 rows of x and of the weights, 2^36 weights, 2^35 outputs, 2^37 numbers of x."""
    most = 1 << 25

    def of(m, n, k):
        return taken(weights(n, k, data=1 << 20), scales(n, k), rows(m, k, data=1 << 45), rows(m, n, data=1 << 50))

    assert of(most, 1, 128) and not of(most + 1, 1, 128)
    assert of(1, most, 128) and not of(1, most + 1, 128)
    assert of(1, most, 2048) and not of(1, most, 2049)
    assert of(1024, most, 1) and not of(1025, most, 1)
    assert of(most, 1, 4096) and not of(most, 1, 4097)
    assert not of(1, 1, (1 << 31) - 1)


def test_other_operations_do_not_take_f8():
    lib = sdhip.load()
    w, x = weights(320, 320), rows(320, 320)
    assert not lib.sdhip_mul_mat_supported(w, x, x)
    assert not lib.sdhip_mul_mat_supported(x, w, x)
    assert not lib.sdhip_norm_supported(w, w)
    assert not lib.sdhip_group_norm_supported(w, w, 4)
    assert not lib.sdhip_attention_supported(x, w, w, x, 0.0, 0.0)
    assert not lib.sdhip_conv2d_supported(w, x, x, sdhip.conv_params())


def test_descriptors_of_f8():
    d = sdhip.desc(torch.zeros((70, 32), dtype=torch.uint8).view(torch.float8_e4m3fn)[:, 3:20])
    assert d.type == F8 and list(d.ne) == [17, 70, 1, 1] and list(d.nb[:2]) == [1, 32]


# ---------------------------------------------------------------- rotary positions


def axes(dims=(32, 32), base=10000.0, order=0, shared=0):
    a = sdhip.RopeAxes()
    a.count, a.order, a.shared = len(dims), order, shared
    for i, d in enumerate(dims[:4]):
        a.dims[i], a.base[i] = d, base
    return a


def norm(kind=sdhip.ROW_NORM_RMS, weight=None, bias=None):
    r = sdhip.RowNorm()
    r.kind, r.eps = kind, 1e-6
    r._held = (weight, bias)
    if weight is not None:
        r.weight = ctypes.pointer(weight)
    if bias is not None:
        r.bias = ctypes.pointer(bias)
    return r


def rope_taken(x, n, at, ax, y):
    return bool(sdhip.load().sdhip_rope_supported(x, n, at, ax, y))


X, Y, AT = rows(2, 3, 7, 64), rows(2, 3, 7, 64, data=2 * FAKE), rows(7, 2, data=3 * FAKE)


def test_rope_taken():
    assert rope_taken(X, None, AT, axes(), Y)
    assert rope_taken(X, None, AT, axes(), X)                                         # in place
    assert rope_taken(X, None, AT, axes(), rows(2, 3, 7, 64, data=2 * FAKE, type=F16))
    for ax in (axes((64,)), axes((2,)), axes((16, 16, 16, 16)), axes(order=1, shared=1)):
        assert rope_taken(X, None, rows(7, ax.count, data=3 * FAKE), ax, Y)
    for at in (rows(1, 2, data=3 * FAKE), rows(2, 1, 7, 2, data=3 * FAKE), rows(2, 1, 1, 2, data=3 * FAKE)):
        assert rope_taken(X, None, at, axes(), Y)
    for w in (rows(64, data=9 * FAKE), rows(1, data=9 * FAKE), rows(3, 1, 64, data=9 * FAKE), rows(2, 3, 7, 64, data=9 * FAKE)):
        assert rope_taken(X, norm(weight=w), AT, axes(), Y) and rope_taken(X, norm(0, bias=w), AT, axes(), Y)
    assert rope_taken(rows(512), None, rows(1, 2, data=3 * FAKE), axes(), rows(512, data=9 * FAKE))
    x = changed(X, "nb", 3, 0)
    assert rope_taken(x, None, AT, axes(), Y)                                         # read: rows may share memory


def test_rope_refused():
    lib = sdhip.load()
    half = rows(2, 3, 7, 64, type=F16)
    bad = [(None, None, AT, axes(), Y), (X, None, None, axes(), Y), (X, None, AT, None, Y), (X, None, AT, axes(), None),
           (half, None, AT, axes(), Y), (half, None, AT, axes(), half)]
    for ax in (axes(()), axes((2,) * 5), axes((33, 31)), axes((32, 34)), axes((32, 0)), axes((64, -2)), axes(base=0.0), axes(base=-1.0),
               axes(base=float("inf")), axes(base=float("nan")), axes(order=2), axes(order=-1)):
        bad.append((X, None, rows(7, max(ax.count, 1), data=3 * FAKE), ax, Y))
    for f, k, v in (("type", 0, F8), ("ne", 0, 63), ("ne", 0, 0), ("ne", 1, 8), ("ne", 2, 0), ("ne", 3, 1), ("nb", 0, 8), ("nb", 1, 6),
                    ("nb", 2, 2), ("nb", 3, 1), ("data", 0, 4 * FAKE + 2)):
        bad += [(changed(X, f, k, v), None, AT, axes(), Y), (X, None, AT, axes(), changed(Y, f, k, v))]
    for f, k, v in (("type", 0, F16), ("ne", 0, 1), ("ne", 1, 6), ("ne", 2, 3), ("ne", 3, 3), ("nb", 0, 8), ("nb", 1, 6),
                    ("data", 0, 3 * FAKE + 1)):
        bad.append((X, None, changed(AT, f, k, v), axes(), Y))
    for n in (norm(3), norm(-1), norm(weight=rows(63, data=9 * FAKE)), norm(bias=rows(3, 3, 7, 64, data=9 * FAKE)),
              norm(weight=rows(64, data=9 * FAKE, type=F16)), norm(weight=rows(64, data=9 * FAKE + 1))):
        bad.append((X, n, AT, axes(), Y))
    # Strides below 0, which reach before the data; more heads than are counted.
    for k in (1, 2, 3):
        bad += [(changed(X, "nb", k, -256), None, AT, axes(), Y), (X, None, changed(AT, "nb", k, -8), axes(), Y)]
        bad += [(X, f(changed(rows(2, 3, 7, 64, data=9 * FAKE), "nb", k, -256)), AT, axes(), Y) for f in (lambda w: norm(weight=w), lambda b: norm(bias=b))]
    many = (1 << 24) + 1
    bad.append((rows(many, 1, 2), None, rows(1, 1, data=1 << 41), axes((2,)), rows(many, 1, 2, data=1 << 40)))
    # What is written over what is read, or over itself.
    bad += [(X, None, AT, axes(), rows(2, 3, 7, 64, data=FAKE + 4)), (X, None, AT, axes(), rows(2, 3, 7, 64, data=3 * FAKE - 256)),
            (X, None, AT, axes(), changed(Y, "nb", 1, 4 * 63)), (X, None, AT, axes(), changed(Y, "nb", 3, 0)),
            (X, norm(weight=rows(64, data=2 * FAKE + 256)), AT, axes(), Y), (X, norm(bias=rows(64, data=FAKE)), AT, axes(), X),
            (X, None, AT, axes(), rows(2, 3, 7, 64, type=F16))]
    wide = rows(514), rows(514, data=9 * FAKE)
    bad.append((wide[0], None, rows(1, 2, data=3 * FAKE), axes(), wide[1]))
    for d in bad:
        assert not rope_taken(*d)
        assert lib.sdhip_rope(*d, None) == sdhip.UNSUPPORTED
    for d in ((changed(X, "data", 0, None), None, AT, axes(), Y), (X, None, changed(AT, "data", 0, None), axes(), Y),
              (X, norm(weight=rows(64, data=None)), AT, axes(), Y), (X, None, AT, axes(), changed(Y, "data", 0, None))):
        assert lib.sdhip_rope(*d, None) == sdhip.ERROR


def test_axes_of_the_front_end():
    a = sdhip.rope_axes([16, 56], [100.0, 5.0], "halves", True)
    assert (a.count, a.order, a.shared, list(a.dims[:2]), list(a.base[:2])) == (2, 1, 1, [16, 56], [100.0, 5.0])
    with pytest.raises(ValueError):
        sdhip.rope_axes([2] * 5)
    with pytest.raises(ValueError):
        sdhip.rope_axes([2, 2], [1.0])
    with pytest.raises(KeyError):
        sdhip.rope_axes([2], order="other")


# ---------------------------------------------------------------- group norm, channels last


def norm_taken(x, y, groups=8):
    return bool(sdhip.load().sdhip_group_norm_last_supported(x, y, groups))


I, J = rows(2, 5, 7, 64), rows(2, 5, 7, 64, data=2 * FAKE)


def wide(data, channels=64, more=16, n=2, h=5, w=7):
    row = 4 * (channels + more)
    return sdhip.view_desc(data, F32, [channels, w, h, n], [4, row, row * w, row * w * h + 64])


def test_group_norm_taken():
    lib = sdhip.load()
    for groups in (1, 3, 8, 64, 65, 1 << 30):
        assert norm_taken(I, J, groups) and norm_taken(I, I, groups)
    assert norm_taken(wide(FAKE), J) and norm_taken(I, wide(4 * FAKE)) and norm_taken(wide(FAKE), wide(FAKE))
    assert norm_taken(changed(I, "nb", 3, 0), J)                                       # read: images may share memory
    assert norm_taken(rows(64), rows(64, data=2 * FAKE)) and norm_taken(rows(9, 64), rows(9, 64, data=2 * FAKE))
    big = rows(1, 1024, 1024, 128, data=1 << 33)
    assert 0 < lib.sdhip_group_norm_last_work_size(big, big, 32) < 1 << 22


def test_group_norm_refused():
    lib = sdhip.load()
    bad = [(None, J, 8), (I, None, 8), (I, J, 0), (I, J, -1)]
    for f, k, v in (("type", 0, F16), ("type", 0, F8), ("ne", 0, 63), ("ne", 1, 0), ("ne", 2, 6), ("ne", 3, 3), ("nb", 0, 8),
                    ("nb", 1, 258), ("nb", 2, 7 * 256 + 4), ("nb", 3, 2), ("nb", 3, -64), ("data", 0, 8 * FAKE + 2)):
        bad += [(changed(I, f, k, v), J, 8), (I, changed(J, f, k, v), 8)]
    bad += [(I, rows(2, 5, 7, 64, data=FAKE + 256), 8), (wide(FAKE), I, 8),
            (I, sdhip.view_desc(2 * FAKE, F32, [64, 7, 5, 2], [4, 252, 252 * 7, 252 * 35]), 8), (I, changed(J, "nb", 3, 0), 8)]
    bad.append((rows((1 << 24) + 1), rows((1 << 24) + 1, data=1 << 40), 8))
    huge = rows(1 << 12, 1 << 10, 1 << 10, 1 << 9)
    bad.append((huge, huge, 8))
    for d in bad:
        assert not norm_taken(*d)
        assert lib.sdhip_group_norm_last(*d, 1e-5, None, None, 0, None) == sdhip.UNSUPPORTED
        assert lib.sdhip_group_norm_last_work_size(*d) == 0
    chain = sdhip.Epilogue()
    redirect = rows(2, 5, 7, 64, data=9 * FAKE)
    chain.redirect = ctypes.pointer(redirect)
    assert lib.sdhip_group_norm_last(I, J, 8, 1e-5, chain, None, 0, None) == sdhip.UNSUPPORTED
    none = changed(I, "data", 0, None)
    assert lib.sdhip_group_norm_last(none, J, 8, 1e-5, None, None, 0, None) == sdhip.ERROR
    big = rows(1, 1024, 1024, 128, data=1 << 33)
    assert lib.sdhip_group_norm_last(big, big, 32, 1e-5, None, None, 0, None) == sdhip.ERROR
    assert b"work" in lib.sdhip_last_error()


@pytest.mark.parametrize("shape,groups", [((3, 69, 565, 960), 32), ((3, 1, 100003, 64), 32), ((1, 1, 263001, 12), 3), ((2, 300, 701, 320), 32),
                                          ((1, 1024, 1024, 128), 32), ((5, 333, 77, 512), 32)])
def test_no_part_of_an_image_is_empty(shape, groups):
    """As many chunks of its pixels as the work buffer holds sums of: the last begins before their end."""
    n, h, w, c = shape
    x = rows(*shape, data=1 << 40)
    sums = sdhip.load().sdhip_group_norm_last_work_size(x, x, groups) // (8 * n * groups)
    parts = (sums - 1) // 2 if (sums - 1) // 2 <= 256 else (sums - 3) // 2
    assert parts > 1 and (parts - 1) * -(-h * w // parts) < h * w
