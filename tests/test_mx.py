"""Argument checks of the microscaled operators, on the CPU: instantllm_amd/csrc/ill_mx_check.h compiled with the host compiler,
the library's and the binding's refusals that need no GPU, and the restatement that the GPU tests compare with."""
from __future__ import annotations

import ctypes as C
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

from instantllm_amd import mx
from instantllm_amd.engine import ILL_E_ARG, ILL_E_FORMAT, ILL_OK, IllError
from oracle import mx as O

CSRC = Path(__file__).resolve().parents[1] / "instantllm_amd" / "csrc"
P = 0x10000   # an address aligned to 16 bytes; never followed here
F32, F16, BF16, MXF8, MXF4 = 0, 1, 2, 8, 16


@pytest.fixture(scope="module")
def checks(tmp_path_factory):
    cxx = shutil.which("g++")
    if not cxx:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("mx")
    (d / "c.cpp").write_text("""
#include <cstdarg>
#include <cstdio>
static int fail(int code, const char* fmt, ...) {
  char text[512]; va_list ap; va_start(ap, fmt); vsnprintf(text, sizeof text, fmt, ap); va_end(ap);
  return code;
}
#include "ill_mx_check.h"
extern "C" {
int rows(int f, int t, void* x, int64_t s, int64_t r, int64_t c, void* codes, void* powers) { return illm::check_rows(f, t, x, s, r, c, codes, powers); }
int product(int f, void* x, void* xp, void* w, void* wp, float* b, void* y, int64_t s, int t, int64_t r, int64_t c, int64_t k) {
  return illm::check_product(f, x, xp, w, wp, b, y, s, t, r, c, k); }
}
""")
    subprocess.run([cxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}", str(d / "c.cpp"), "-o", str(d / "c.so")], check=True)
    lib = C.CDLL(str(d / "c.so"))
    A, L, I = C.c_void_p, C.c_int64, C.c_int
    lib.rows.argtypes = [I, I, A, L, L, L, A, A]
    lib.product.argtypes = [I, A, A, A, A, A, A, L, I, L, L, L]
    return lib


ROWS = dict(format=MXF8, dtype=F16, x=P, stride=896, rows=5, cols=896, codes=P, powers=P)


@pytest.mark.parametrize("kw,code", [
    ({}, ILL_OK), (dict(format=MXF4, dtype=F32, stride=900), ILL_OK), (dict(rows=0, x=None, codes=None), ILL_OK), (dict(cols=32, stride=32, rows=1 << 29), ILL_OK),
    (dict(format=0), ILL_E_FORMAT), (dict(format=9), ILL_E_FORMAT), (dict(dtype=3), ILL_E_FORMAT), (dict(dtype=MXF8), ILL_E_FORMAT),
    (dict(cols=0, stride=0), ILL_E_ARG), (dict(cols=48), ILL_E_ARG), (dict(cols=-32), ILL_E_ARG), (dict(rows=-1), ILL_E_ARG),
    (dict(rows=1 << 30), ILL_E_ARG), (dict(rows=1 << 62), ILL_E_ARG), (dict(stride=895), ILL_E_ARG), (dict(stride=900), ILL_E_ARG), (dict(stride=1 << 40), ILL_E_ARG),
    (dict(x=None), ILL_E_ARG), (dict(x=P + 8), ILL_E_ARG), (dict(codes=None), ILL_E_ARG), (dict(powers=None), ILL_E_ARG), (dict(codes=P + 4), ILL_E_ARG),
    (dict(powers=P + 1), ILL_E_ARG)])
def test_rows_are_checked(checks, kw, code):
    assert checks.rows(*{**ROWS, **kw}.values()) == code


PRODUCT = dict(format=MXF8, x=P, xp=P, w=P, wp=P, bias=None, y=P, stride=1152, dtype=F16, rows=3, cols=1152, inner=896)


@pytest.mark.parametrize("kw,code", [
    ({}, ILL_OK), (dict(format=MXF4, dtype=F32, bias=P, stride=1153, y=P + 4), ILL_OK), (dict(rows=0, x=None, y=None), ILL_OK), (dict(cols=1, stride=1, y=P + 2), ILL_OK),
    (dict(format=F16), ILL_E_FORMAT), (dict(dtype=MXF4), ILL_E_FORMAT), (dict(inner=0), ILL_E_ARG), (dict(inner=100), ILL_E_ARG), (dict(inner=1 << 21), ILL_E_ARG),
    (dict(cols=0), ILL_E_ARG), (dict(cols=1 << 25, stride=1 << 25), ILL_E_ARG), (dict(rows=-1), ILL_E_ARG), (dict(rows=1 << 27), ILL_E_ARG),
    (dict(rows=1 << 22), ILL_E_ARG), (dict(stride=1151), ILL_E_ARG), (dict(y=None), ILL_E_ARG), (dict(y=P + 1), ILL_E_ARG), (dict(y=P + 2, dtype=F32), ILL_E_ARG),
    (dict(bias=P + 2), ILL_E_ARG), (dict(x=None), ILL_E_ARG), (dict(xp=None), ILL_E_ARG), (dict(w=None), ILL_E_ARG), (dict(wp=P + 8), ILL_E_ARG), (dict(w=P + 8), ILL_E_ARG)])
def test_products_are_checked(checks, kw, code):
    assert checks.product(*{**PRODUCT, **kw}.values()) == code


def test_binding_refuses():
    with pytest.raises(ValueError, match="format 'mxf6'"):
        mx.quantize(P, P, P, 1, 32, format="mxf6")
    with pytest.raises(ValueError, match="type 'f64'"):
        mx.dequantize(P, P, P, 1, 32, dtype="f64")
    with pytest.raises(ValueError, match="64 bits"):
        mx.product(P, P, P, P, P, 1 << 64, 32, 32)
    assert mx.code_bytes("mxf8", 64) == 64 and mx.code_bytes("mxf4", 64) == 32


def test_library_refuses_without_gpu():
    for call in (lambda: mx.quantize(P, P, P, 1, 33), lambda: mx.dequantize(P, P + 1, P, 1, 32), lambda: mx.product(P, P, P, P, P, 1, 16, 96, y_stride=15)):
        with pytest.raises(IllError, match="mx: ") as e:
            call()
        assert e.value.code == ILL_E_ARG
    mx.quantize(0, 0, 0, 0, 32)   # nothing to do


@pytest.mark.parametrize("fmt", ["mxf8", "mxf4"])
def test_restatement(fmt):
    """Every code comes back as itself, borders go to the even code, sizes past the largest end there."""
    sizes, n = O.SIZES[fmt], {"mxf8": 127, "mxf4": 8}[fmt]
    x = np.zeros((n, 32))
    x[:, 0], x[:, 1] = sizes[-1], sizes
    x[:, 2] = -x[:, 1]
    held, powers = O.quantize(x, fmt)
    codes = O.unpack(held, fmt)
    assert (powers == 127).all() and np.array_equal(codes[:, 1], np.arange(n)) and np.array_equal(codes[:, 2], np.arange(n) + (n + 1 & ~7 if fmt == "mxf8" else 8))
    assert np.array_equal(O.values(held, powers, fmt), x)
    mid = (sizes[1:] + sizes[:-1]) / 2
    x = np.zeros((n - 1, 32))
    x[:, 0], x[:, 1] = sizes[-1], mid
    assert np.array_equal(O.unpack(O.quantize(x, fmt)[0], fmt)[:, 1], [i + (i & 1) for i in range(n - 1)])
    x = np.full((1, 32), 2.0 ** (O.TOP[fmt] + 1) * 0.999)
    held, powers = O.quantize(x, fmt)
    assert powers[0, 0] == 127 and (O.values(held, powers, fmt) == sizes[-1]).all()
    # the least power, zeros, and blocks that hold no value
    for v, byte in ((2.0 ** -149, 0), (0.0, 0), (np.inf, 255), (np.nan, 255), (2.0 ** 127, 254 - O.TOP[fmt])):
        x = np.zeros((1, 32))
        x[0, 7] = v
        assert O.quantize(x, fmt)[1][0, 0] == byte
