"""SiLU as the channels-last norms' outputs take it (`fast_silu` of norm_last.hip),
compiled from its own text for the host, the hardware's power of two and
reciprocal by the host's: its whole range against 64 bits.

Bound: with exp(-x) past 1 that power, its correction, the sum with 1, the
reciprocal and the product are rounded once each, 5 roundings of 2^-24; what the
correction leaves out is its square, 2^-36, and the 6th covers it.  From -87.33
on the sum passes 2^126 and its reciprocal may be rounded to a 0: |x| 2^-126."""

import ctypes
import os
import re
import subprocess

import numpy as np
import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "stable-diffusion.assembly_amd", "csrc",
                      "norm_last.hip")

HOST = """
#include <cmath>
#define __device__
#define __forceinline__ inline
static float host_rcp(float v) { return 1.0f / v; }
#define __builtin_amdgcn_exp2f exp2f
#define __builtin_amdgcn_rcpf host_rcp
%s
extern "C" void silu_of(const float *x, float *y, long n) {
    for (long i = 0; i < n; ++i) y[i] = fast_silu(x[i]);
}
"""


@pytest.fixture(scope="module")
def fast_silu(tmp_path_factory):
    with open(SOURCE) as f:
        body = re.search(r"^__device__ __forceinline__ float fast_silu\(float x\) \{.*?^\}", f.read(), re.S | re.M).group(0)
    folder = tmp_path_factory.mktemp("silu")
    (folder / "silu.cpp").write_text(HOST % body)
    subprocess.run(["g++", "-O1", "-mfma", "-ffp-contract=off", "-shared", "-fPIC", str(folder / "silu.cpp"), "-o",
                    str(folder / "silu.so")], check=True, timeout=120)
    lib = ctypes.CDLL(str(folder / "silu.so"))

    def call(x):
        x = np.ascontiguousarray(x, np.float32)
        y = np.empty_like(x)
        at = ctypes.POINTER(ctypes.c_float)
        lib.silu_of(x.ctypes.data_as(at), y.ctypes.data_as(at), ctypes.c_long(x.size))
        return x, y

    return call


def within(x, y):
    x64 = x.astype(np.float64)
    with np.errstate(over="ignore"):
        want = x64 / (1.0 + np.exp(-x64))
    err = 6 * 2.0 ** -24 * np.abs(want) + 2.0 ** -126 * np.where(x64 < -87.3, np.abs(x64), 1.0)
    return np.abs(y - want) <= err  # False of a NaN


@pytest.mark.parametrize("low,high", [(-130.0, -80.0), (-20.0, 20.0), (-2000.0, 2000.0), (-1e5, 1e5), (80.0, 130.0), (-3.4e38, 3.4e38)])
def test_ranges(fast_silu, low, high):
    x, y = fast_silu(np.linspace(low, high, 1 << 20))
    good = within(x, y)
    assert good.all(), (x[~good][:5], y[~good][:5])


def test_every_float_where_the_power_overflows(fast_silu):
    """From -88.5 to -89.5, -log2(e) x passes 2^128's 128."""
    first, last = (np.float32(v).view(np.uint32) for v in (-88.5, -89.5))
    x, y = fast_silu(np.arange(first, last, dtype=np.uint32).view(np.float32))
    good = within(x, y)
    assert good.all(), (x[~good][:5], y[~good][:5])


def test_ends(fast_silu):
    """The greatest numbers, an infinity and a NaN: themselves, or 0."""
    greatest = np.finfo(np.float32).max
    _, y = fast_silu([2.3e38, 2.5e38, greatest, np.inf, -2.3e38, -2.5e38, -greatest, 0.0, -0.0])
    assert y[:4].tolist() == [np.float32(2.3e38), np.float32(2.5e38), greatest, np.inf]
    assert (y[4:] == 0).all()
    assert np.isnan(fast_silu([np.nan])[1]).all()
