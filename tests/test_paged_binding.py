"""The Python binding of the paged-cache operators, on the CPU: numbers that do not fit their C types are refused, not cut off."""
from __future__ import annotations

import ctypes as C

import pytest

from instantllm_amd.engine import ILL_E_ARG, IllError
from instantllm_amd.paged import Batch, PagedAttention

P16 = 0x10000


class Calls:
    """A library that notes the numbers of a call as C sees them."""
    def __init__(self):
        self.got = []

    def ill_last_error(self):
        return b"refused"

    def ill_paged_attend(self, h, batch, q, qs, k, v, window, sinks, out, os, dtype, stream):
        self.got = [C.c_int64(qs).value, C.c_int(window).value, C.c_int(sinks).value, C.c_int64(os).value]
        return ILL_E_ARG if min(self.got) < 0 else 0

    def ill_paged_append(self, *a):
        return 0


@pytest.fixture()
def op():
    p = PagedAttention.__new__(PagedAttention)
    p.h, p.lib, p.type, p.q_width, p.kv_width = None, Calls(), 1, 896, 128
    return p


def test_batch_fields(op):
    b = op.batch(P16, 2 * P16, 5, 40, 3, rows=7, row0=3 * P16, max_rows=4, table_stride=9)
    assert isinstance(b, Batch)
    assert [getattr(b, n) for n, _ in Batch._fields_] == [3, 5, 9, 7, 4, 40, P16, 2 * P16, 3 * P16]
    b = op.batch(P16, 2 * P16, 5, 40, 3)
    assert [getattr(b, n) for n, _ in Batch._fields_] == [3, 5, 5, 3, 0, 40, P16, 2 * P16, None]


@pytest.mark.parametrize("kw", [dict(seqs=1 << 32), dict(seqs=(1 << 32) + 3), dict(table_width=(1 << 32) + 5), dict(rows=(1 << 64) + 3), dict(pages=(1 << 64) + 40),
                                dict(max_rows=1 << 63), dict(table_stride=-(1 << 63) - 1), dict(lens=1 << 64)])
def test_batch_numbers_that_do_not_fit(op, kw):
    good = dict(lens=P16, table=P16, table_width=5, pages=40, seqs=3)
    op.batch(**good)
    with pytest.raises(ValueError):
        op.batch(**{**good, **kw})


@pytest.mark.parametrize("kw", [dict(window=(1 << 32) + 5), dict(window=1 << 31), dict(sinks=1 << 32), dict(window=-(1 << 32)), dict(q_stride=(1 << 64) + 896),
                                dict(out_stride=(1 << 64) + 896)])
def test_attend_numbers_that_do_not_fit(op, kw):
    b = op.batch(P16, P16, 5, 40, 3)
    with pytest.raises(ValueError):
        op.attend(b, P16, P16, P16, 2 * P16, **kw)
    assert op.lib.got == []


def test_attend_numbers_that_fit(op):
    b = op.batch(P16, P16, 5, 40, 3)
    op.attend(b, P16, P16, P16, 2 * P16, window=(1 << 31) - 1, sinks=7, q_stride=1 << 40)
    assert op.lib.got == [1 << 40, (1 << 31) - 1, 7, 896]
    with pytest.raises(IllError):   # the library's own refusal
        op.attend(b, P16, P16, P16, 2 * P16, window=-1)
    assert op.lib.got == [896, -1, 0, 896]


def test_append_numbers_that_do_not_fit(op):
    b = op.batch(P16, P16, 5, 40, 3)
    op.append(b, P16, P16, P16, P16, x_stride=1152)
    for kw in (dict(x_stride=(1 << 64) + 1152), dict(k_stride=1 << 63), dict(bias=1 << 64)):
        with pytest.raises(ValueError):
            op.append(b, P16, P16, P16, P16, **kw)


@pytest.mark.parametrize("kw", [dict(page_size=(1 << 32) + 16), dict(streams=1 << 32), dict(rotary_dim=(1 << 32) + 64), dict(strides=((1 << 64) + 2048, 128, 64))])
def test_descriptions_that_do_not_fit(kw):
    with pytest.raises(ValueError, match="bits"):
        PagedAttention(14, 2, 64, **kw)
