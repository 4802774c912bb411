"""The 8-bit floating-point products whose chain or gated GELU is computed apart
(fuse = 0) refuse what the fused form refuses, before anything is launched."""

import ctypes

import pytest

import sdhip
from test_image_operators import FAKE, rows, scales, weights

W, S, X, Y = weights(320, 320), scales(320, 320), rows(40, 320), rows(40, 320, data=1 << 40)


@pytest.fixture(params=["", "fuse=0", "fuse_residual=0"])
def tuned(request):
    sdhip.load()
    sdhip.set_tuning(request.param + ("," if request.param else "") + "f8_form=1")  # without a work buffer
    yield
    sdhip.set_tuning("")


@pytest.mark.parametrize("data,message", [(None, b"without data"), ((1 << 42) + 2, b"no multiple of 4")])
def test_gated_output(tuned, data, message):
    lib = sdhip.load()
    assert lib.sdhip_mul_mat_f8_gated(W, S, X, Y, None, rows(40, 160, data=data), None, 0, None) == sdhip.ERROR
    assert message in lib.sdhip_last_error()


def test_redirect(tuned):
    lib = sdhip.load()
    e, at = sdhip.Epilogue(), rows(40, 320, data=(1 << 42) + 2)
    e.count, e.from_redirect, e.redirect = 0, 1, ctypes.pointer(at)
    assert lib.sdhip_mul_mat_f8(W, S, X, Y, e, None, 0, None) == sdhip.ERROR
    assert b"no multiple of 4" in lib.sdhip_last_error()
