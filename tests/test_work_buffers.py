"""The front end's `work`: a buffer that is smaller than its call needs is refused
by its own bytes, whatever the call needed when it was made; one of other numbers
than bytes counts as what it holds.  Without a device: what is refused is refused
before a launch."""

import ctypes

import pytest
import torch

import sdhip


@pytest.fixture(autouse=True)
def no_stream(monkeypatch):
    monkeypatch.setattr(sdhip, "stream_handle", lambda: ctypes.c_void_p(None))
    sdhip.load()
    yield
    sdhip.set_tuning("")


def f8(m=40, k=256, n=128):
    w = torch.zeros((n, k), dtype=torch.uint8).view(torch.float8_e4m3fn)
    return w, torch.ones((1, 2)), torch.zeros((m, k)), torch.empty((m, n))


def calls():
    """{name: (tuning, call of a work buffer)}, each of which needs one."""
    w, s, x, y = f8()
    out = torch.empty((40, 64))
    image = torch.zeros((1, 64, 64, 64))
    q4 = torch.zeros((128, 8, 18), dtype=torch.uint8)
    planes, kernel = torch.zeros((1, 32, 40, 40)), torch.zeros((32, 32, 3, 3), dtype=torch.float16)
    wh, xh, yh = torch.zeros((64, 1024), dtype=torch.float16), torch.zeros((16, 1024)), torch.empty((16, 64))
    q = torch.zeros((1, 1, 512, 320))
    return {
        "mul_mat_f8": ("f8_form=3", lambda b: sdhip.mul_mat_f8(w, s, x, y, work=b)),
        "mul_mat_f8_gated": ("f8_form=3", lambda b: sdhip.mul_mat_f8_gated(w, s, x, y, out, work=b)),
        "group_norm_last": ("", lambda b: sdhip.group_norm_last(image, torch.empty_like(image), 32, 1e-5, work=b)),
        "mul_mat": ("q4_form=3", lambda b: sdhip.mul_mat(q4, x, y, work=b)),
        "mul_mat split": ("", lambda b: sdhip.mul_mat(wh, xh, yh, work=b)),
        "mul_mat_gated": ("q4_form=3", lambda b: sdhip.mul_mat_gated(q4, x, y, out, work=b)),
        "conv2d": ("", lambda b: sdhip.conv2d(kernel, planes, torch.empty((1, 32, 40, 40)), sdhip.conv_params(1, 1, 1, 1), work=b)),
        "attention": ("", lambda b: sdhip.attention(q, q, q, torch.empty((1, 512, 1, 320)), 1.0, work=b)),
        "group_norm": ("", lambda b: sdhip.group_norm(torch.zeros((1, 64, 64, 64)), torch.empty((1, 64, 64, 64)), 32, 1e-5, work=b)),
    }


@pytest.mark.parametrize("name", calls())
@pytest.mark.parametrize("held", [torch.empty(16, dtype=torch.uint8), torch.empty(4)])
def test_a_smaller_buffer_is_refused(name, held):
    text, call = calls()[name]
    sdhip.set_tuning(text)
    with pytest.raises(Exception, match="work buffer of 16 bytes"):
        call(held)


def test_a_buffer_of_another_form():
    """Made for the few rows' form, which needs none, or for fewer rows."""
    w, s, x, y = f8(200)
    sdhip.set_tuning("f8_form=3")
    size = sdhip.load().sdhip_mul_mat_f8_work_size(*(sdhip.desc(t) for t in f8(40)))
    assert 0 < size < sdhip.load().sdhip_mul_mat_f8_work_size(*(sdhip.desc(t) for t in (w, s, x, y)))
    with pytest.raises(Exception, match=f"work buffer of {size} bytes"):
        sdhip.mul_mat_f8(w, s, x, y, work=torch.empty(size, dtype=torch.uint8))


def test_numbers_apart_are_no_buffer():
    """Every second number, or one number many times, holds fewer bytes than it has numbers of."""
    w, s, x, y = f8()
    sdhip.set_tuning("f8_form=3")
    for held in (torch.empty(1 << 20)[::2], torch.empty(1).expand(1 << 20)):
        with pytest.raises(ValueError, match="contiguous"):
            sdhip.mul_mat_f8(w, s, x, y, work=held)
