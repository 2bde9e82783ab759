"""Argument checks of the paged-cache operators, on the CPU: instantllm_amd/csrc/ill_paged_check.h compiled with the host
compiler and called with the binding's structures, and the library's own refusals that need no GPU."""
from __future__ import annotations

import ctypes as C
import shutil
import subprocess
from pathlib import Path

import pytest

from instantllm_amd.engine import ILL_E_ARG, ILL_E_FORMAT, IllError
from instantllm_amd.paged import Batch, PagedAttention, _Desc, _Rows

CSRC = Path(__file__).resolve().parents[1] / "instantllm_amd" / "csrc"
P16 = 0x10000   # an address aligned to 16 bytes; never followed here


@pytest.fixture(scope="module")
def checks(tmp_path_factory):
    cxx = shutil.which("g++")
    if not cxx:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("paged")
    (d / "c.cpp").write_text("""
#include <cstdarg>
#include <cstdio>
static char text[512];
static int fail(int code, const char* fmt, ...) {
  va_list ap; va_start(ap, fmt); vsnprintf(text, sizeof text, fmt, ap); va_end(ap);
  return code;
}
#include "ill_paged_check.h"
extern "C" {
const char* message() { return text; }
int desc(ill_paged_desc* d) { return illp::check_desc(*d); }
int append(ill_paged_desc* d, ill_paged_batch* b, ill_paged_rows* x, void* k, void* v) { return illp::check_append(*d, b, x, k, v); }
int attend(ill_paged_desc* d, ill_paged_batch* b, void* q, int64_t qs, void* k, void* v, int w, int s, void* o, int64_t os, int t) {
  return illp::check_attend(*d, b, q, qs, k, v, w, s, o, os, t); }
}
""")
    subprocess.run([cxx, "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}", str(d / "c.cpp"), "-o", str(d / "c.so")], check=True)
    lib = C.CDLL(str(d / "c.so"))
    P, L, I = C.c_void_p, C.c_int64, C.c_int
    lib.attend.argtypes = [P, P, P, L, P, P, I, I, P, L, I]
    lib.append.argtypes = [P, P, P, P, P]
    lib.message.restype = C.c_char_p
    return lib


def _desc(**kw):
    d = dict(dtype=1, heads=14, kv_heads=2, head_dim=64, page_size=16, rotary_dim=64, rope_base=1e6, norm_eps=1e-6)
    d.update(kw)
    return _Desc(**d)


def _batch(**kw):
    b = dict(seqs=3, table_width=5, table_stride=8, rows=3, max_rows=0, pages=40, lens=P16, table=P16, row0=None)
    b.update(kw)
    return Batch(**b)


def _rows(**kw):
    x = dict(q=P16, k=P16, v=P16, q_out=2 * P16, q_stride=1152, k_stride=1152, v_stride=1152, q_out_stride=896, dtype=1)
    x.update(kw)
    return _Rows(**x)


def test_description_defaults(checks):
    d = _desc()
    assert checks.desc(C.byref(d)) == 0
    assert (d.page_stride, d.slot_stride, d.head_stride) == (16 * 128, 128, 64)
    assert d.scale == 0.125
    d = _desc(page_stride=2 * 16 * 64, slot_stride=64, head_stride=16 * 64)   # heads outside positions
    assert checks.desc(C.byref(d)) == 0


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=0), ILL_E_FORMAT), (dict(dtype=3), ILL_E_FORMAT), (dict(heads=13), ILL_E_ARG), (dict(kv_heads=0), ILL_E_ARG),
    (dict(heads=1), ILL_E_ARG), (dict(heads=2048), ILL_E_ARG), (dict(head_dim=80), ILL_E_ARG), (dict(page_size=8), ILL_E_ARG),
    (dict(page_size=24), ILL_E_ARG), (dict(page_size=2048), ILL_E_ARG), (dict(rotary_dim=24), ILL_E_ARG), (dict(rotary_dim=80), ILL_E_ARG),
    (dict(rotary_dim=-16), ILL_E_ARG), (dict(rope_base=0.0), ILL_E_ARG), (dict(rope_base=float("nan")), ILL_E_ARG), (dict(norm_eps=-1.0), ILL_E_ARG),
    (dict(scale=-1.0), ILL_E_ARG), (dict(scale=float("inf")), ILL_E_ARG), (dict(page_stride=2048), ILL_E_ARG),
    (dict(page_stride=2052, slot_stride=128, head_stride=64), ILL_E_ARG), (dict(page_stride=2048, slot_stride=64, head_stride=64), ILL_E_ARG),
    (dict(page_stride=2048, slot_stride=1 << 62, head_stride=64), ILL_E_ARG)])
def test_descriptions_refused(checks, kw, code):
    d = _desc(**kw)
    assert checks.desc(C.byref(d)) == code
    assert checks.message().startswith(b"paged: ")


@pytest.mark.parametrize("kw", [
    dict(seqs=-1), dict(rows=-1), dict(rows=2), dict(rows=1 << 27), dict(rows=(1 << 26) // 14 + 1),
    dict(seqs=(1 << 22) // 14 + 1, rows=1 << 20), dict(seqs=1 << 30, rows=1 << 30), dict(table_width=0), dict(table_stride=4),
    dict(table_width=1 << 27, table_stride=1 << 27), dict(pages=0), dict(pages=1 << 31), dict(max_rows=-1), dict(lens=None), dict(table=None),
    dict(lens=P16 + 2), dict(row0=P16 + 1)])
def test_batches_refused(checks, kw):
    d, b, x = _desc(), _batch(), _rows()
    checks.desc(C.byref(d))
    assert checks.append(C.byref(d), C.byref(b), C.byref(x), P16, P16) == 0
    assert checks.attend(C.byref(d), C.byref(b), P16, 896, P16, P16, 0, 0, 2 * P16, 896, 1) == 0
    b = _batch(**kw)
    assert checks.append(C.byref(d), C.byref(b), C.byref(x), P16, P16) == ILL_E_ARG
    assert checks.attend(C.byref(d), C.byref(b), P16, 896, P16, P16, 0, 0, 2 * P16, 896, 1) == ILL_E_ARG


def test_pages_that_overlap_are_refused(checks):
    """Heads outermost, [kv][pages][slots][dim]: as many pages as lie between two heads."""
    d, x = _desc(page_stride=1024, slot_stride=64, head_stride=40 * 1024), _rows()
    assert checks.desc(C.byref(d)) == 0
    for pages, rc in ((40, 0), (41, ILL_E_ARG)):
        b = _batch(pages=pages)
        assert checks.append(C.byref(d), C.byref(b), C.byref(x), P16, P16) == rc


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=2), ILL_E_FORMAT), (dict(dtype=7), ILL_E_FORMAT), (dict(k=None), ILL_E_ARG), (dict(v=None), ILL_E_ARG), (dict(q_out=None), ILL_E_ARG),
    (dict(q=P16 + 8), ILL_E_ARG), (dict(k=P16 + 2), ILL_E_ARG), (dict(q_out=P16 + 4), ILL_E_ARG), (dict(q_stride=888), ILL_E_ARG),
    (dict(k_stride=1156), ILL_E_ARG), (dict(v_stride=120), ILL_E_ARG), (dict(q_out_stride=900), ILL_E_ARG), (dict(q_stride=1 << 40), ILL_E_ARG),
    (dict(bias=P16 + 2), ILL_E_ARG), (dict(q_norm=P16 + 1), ILL_E_ARG), (dict(positions=P16 + 3), ILL_E_ARG), (dict(q_out=P16), ILL_E_ARG),
    (dict(q_out=P16, q_stride=896, q_out_stride=896, dtype=0), ILL_E_ARG)])
def test_rows_refused(checks, kw, code):
    d, b, x = _desc(), _batch(), _rows(**kw)
    checks.desc(C.byref(d))
    assert checks.append(C.byref(d), C.byref(b), C.byref(x), P16, P16) == code
    x = _rows(q=None, q_out=None, q_stride=0, dtype=0)
    assert checks.append(C.byref(d), C.byref(b), C.byref(x), P16, P16) == 0
    for caches in ((None, P16), (P16, P16 + 8)):
        assert checks.append(C.byref(d), C.byref(b), C.byref(x), *caches) == ILL_E_ARG


def test_attend_refused(checks):
    d, b = _desc(), _batch()
    checks.desc(C.byref(d))

    def call(q=P16, qs=896, k=P16, v=P16, w=0, s=0, o=2 * P16, os=896, t=1):
        return checks.attend(C.byref(d), C.byref(b), q, qs, k, v, w, s, o, os, t)
    assert call() == 0 and call(t=0, os=900) == 0 and call(w=5, s=1 << 30) == 0
    for kw in (dict(q=None), dict(q=P16 + 2), dict(qs=890), dict(qs=64), dict(k=None), dict(v=P16 + 4), dict(w=-1), dict(s=-1), dict(o=None),
               dict(o=P16), dict(os=100), dict(os=900), dict(t=0, os=898)):
        assert call(**kw) == ILL_E_ARG, kw
    assert call(t=2) == ILL_E_FORMAT and call(t=9) == ILL_E_FORMAT


def test_library_refuses_without_a_gpu():
    lib_path = CSRC.parent / "libillhip.so"
    if not lib_path.exists():
        pytest.skip("libillhip.so not built")
    with pytest.raises(IllError) as e:
        PagedAttention(14, 2, 80)
    assert e.value.code == ILL_E_ARG and "head size 80" in str(e.value)
    with pytest.raises(ValueError, match="type 'f8'"):
        PagedAttention(14, 2, 64, dtype="f8")
    from instantllm_amd.engine import load_library
    lib = load_library()
    b, x = _batch(), _rows()
    assert lib.ill_paged_append(None, C.byref(b), C.byref(x), P16, P16, None) == ILL_E_ARG
    assert lib.ill_paged_attend(None, C.byref(b), P16, 896, P16, P16, 0, 0, 2 * P16, 896, 1, None) == ILL_E_ARG
    assert lib.ill_paged_create(None, None) == ILL_E_ARG
    assert lib.ill_paged_destroy(None) == 0
