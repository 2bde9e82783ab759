"""Argument checks of paged caches of microscaled values, and of reading rows out of either kind, on the CPU:
instantllm_amd/csrc/ill_paged_check.h compiled with the host compiler, and the binding's own refusals."""
from __future__ import annotations

import ctypes as C
import shutil
import subprocess
from pathlib import Path

import pytest

from instantllm_amd.engine import ILL_E_ARG, ILL_E_FORMAT, ILL_OK, IllError
from instantllm_amd.paged import Batch, PagedAttention, _Desc, _Rows

CSRC = Path(__file__).resolve().parents[1] / "instantllm_amd" / "csrc"
P16 = 0x10000   # an address aligned to 16 bytes; never followed here
F32, F16, BF16, MXF8, MXF4 = 0, 1, 2, 8, 16


@pytest.fixture(scope="module")
def checks(tmp_path_factory):
    cxx = shutil.which("g++")
    if not cxx:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("paged_mx")
    (d / "c.cpp").write_text("""
#include <cstdarg>
#include <cstdio>
static int fail(int code, const char* fmt, ...) {
  char text[512]; va_list ap; va_start(ap, fmt); vsnprintf(text, sizeof text, fmt, ap); va_end(ap);
  return code;
}
#include "ill_paged_check.h"
extern "C" {
int desc(ill_paged_desc* d) { return illp::check_desc(*d); }
int append(ill_paged_desc* d, ill_paged_batch* b, ill_paged_rows* x, void* k, void* v) { return illp::check_append(*d, b, x, k, v); }
int attend(ill_paged_desc* d, ill_paged_batch* b, void* q, int64_t qs, void* k, void* v, int w, int s, void* o, int64_t os, int t) {
  return illp::check_attend(*d, b, q, qs, k, v, w, s, o, os, t); }
int read(ill_paged_desc* d, ill_paged_batch* b, void* kc, void* vc, void* k, int64_t ks, void* v, int64_t vs, int t) {
  return illp::check_read(*d, b, kc, vc, k, ks, v, vs, t); }
}
""")
    subprocess.run([cxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}", str(d / "c.cpp"), "-o", str(d / "c.so")], check=True)
    lib = C.CDLL(str(d / "c.so"))
    P, L, I = C.c_void_p, C.c_int64, C.c_int
    lib.append.argtypes = [P, P, P, P, P]
    lib.attend.argtypes = [P, P, P, L, P, P, I, I, P, L, I]
    lib.read.argtypes = [P, P, P, P, P, L, P, L, I]
    return lib


def _desc(checks, **kw):
    d = _Desc(**{**dict(dtype=F16 | MXF8, heads=14, kv_heads=2, head_dim=64, page_size=16, rotary_dim=64, rope_base=1e6, norm_eps=1e-6), **kw})
    return d, checks.desc(C.byref(d))


def _batch(**kw):
    return Batch(**{**dict(seqs=3, table_width=5, table_stride=8, rows=3, max_rows=0, pages=40, lens=P16, table=P16, row0=None), **kw})


def test_description_defaults(checks):
    d, rc = _desc(checks)
    assert rc == ILL_OK and d.page_stride == 16 * 2 * (64 + 2)
    d, rc = _desc(checks, dtype=BF16 | MXF8, head_dim=128, rotary_dim=0, page_size=1024, kv_heads=7, page_stride=1 << 40)
    assert rc == ILL_OK and d.page_stride == 1 << 40


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=MXF8), ILL_E_FORMAT), (dict(dtype=F16 | MXF4), ILL_E_FORMAT), (dict(dtype=F16 | MXF8 | MXF4), ILL_E_FORMAT), (dict(dtype=3 | MXF8), ILL_E_FORMAT),
    (dict(dtype=F16 | MXF8 | 32), ILL_E_FORMAT), (dict(slot_stride=64), ILL_E_ARG), (dict(head_stride=64), ILL_E_ARG), (dict(page_stride=2111), ILL_E_ARG),
    (dict(page_stride=2096), ILL_E_ARG), (dict(page_stride=2120), ILL_E_ARG), (dict(page_stride=-16), ILL_E_ARG), (dict(page_stride=(1 << 63) - 16), ILL_E_ARG),
    (dict(head_dim=80), ILL_E_ARG), (dict(page_size=8), ILL_E_ARG)])
def test_descriptions_are_checked(checks, kw, code):
    assert _desc(checks, **kw)[1] == code


def test_batches_and_types(checks):
    d, _ = _desc(checks)
    rows = dict(q=P16, k=P16, v=P16, q_out=2 * P16, q_stride=1152, k_stride=1152, v_stride=1152, q_out_stride=896)
    for t, code in ((F16, ILL_OK), (F32, ILL_OK), (BF16, ILL_E_FORMAT), (F16 | MXF8, ILL_E_FORMAT)):
        assert checks.append(C.byref(d), C.byref(_batch()), C.byref(_Rows(**rows, dtype=t)), P16, P16) == code
        assert checks.attend(C.byref(d), C.byref(_batch()), P16, 896, P16, P16, 0, 0, 2 * P16, 896, t) == code
        assert checks.read(C.byref(d), C.byref(_batch()), P16, P16, P16, 128, 2 * P16, 128, t) == code
    far, _ = _desc(checks, page_stride=1 << 58)
    assert checks.attend(C.byref(far), C.byref(_batch(pages=3)), P16, 896, P16, P16, 0, 0, 2 * P16, 896, F16) == ILL_OK
    assert checks.attend(C.byref(far), C.byref(_batch(pages=4)), P16, 896, P16, P16, 0, 0, 2 * P16, 896, F16) == ILL_E_ARG


READ = dict(kc=P16, vc=P16, k=P16, k_stride=128, v=2 * P16, v_stride=128, t=F16)


@pytest.mark.parametrize("dtype", [F16, F16 | MXF8])
@pytest.mark.parametrize("kw,code", [
    ({}, ILL_OK), (dict(t=F32, k_stride=132), ILL_OK), (dict(t=BF16), ILL_E_FORMAT), (dict(kc=None), ILL_E_ARG), (dict(vc=P16 + 8), ILL_E_ARG), (dict(k=None), ILL_E_ARG),
    (dict(v=P16 + 2), ILL_E_ARG), (dict(k_stride=127), ILL_E_ARG), (dict(v_stride=132), ILL_E_ARG), (dict(v=P16), ILL_E_ARG)])
def test_reads_are_checked(checks, dtype, kw, code):
    d, _ = _desc(checks, dtype=dtype)
    assert checks.read(C.byref(d), C.byref(_batch()), *{**READ, **kw}.values()) == code


def test_binding_refuses():
    with pytest.raises(ValueError, match="cache 'mxf4'"):
        PagedAttention(14, 2, 64, cache="mxf4")
    with pytest.raises(ValueError, match="strides are"):
        PagedAttention(14, 2, 64, cache="mxf8", strides=(2048, 64, 1024))
    with pytest.raises(ValueError, match="strides are"):
        PagedAttention(14, 2, 64, page_stride=4096)
    with pytest.raises(ValueError, match="64 bits"):
        PagedAttention(14, 2, 64, cache="mxf8", page_stride=1 << 64)
    with pytest.raises(IllError, match="microscaled pages") as e:
        PagedAttention(14, 2, 64, cache="mxf8", page_stride=2048)
    assert e.value.code == ILL_E_ARG
