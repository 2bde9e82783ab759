"""The most sequences of a batch of the paged-cache operators: every workgroup looks all of them over, so a call's time grows with
their square (16384 sequences of two key/value heads 4 ms; 2^22, which were accepted, some minutes)."""
from __future__ import annotations

import ctypes as C

import pytest

from instantllm_amd.engine import ILL_E_ARG
from test_paged import P16, _batch, _desc, _rows, checks  # noqa: F401


@pytest.mark.parametrize("one_row", [True, False])
@pytest.mark.parametrize("heads,kv,most", [(1, 1, 1 << 14), (14, 2, 1 << 14), (256, 256, 1 << 14), (512, 8, 1 << 13), (1024, 1024, 1 << 12)])
def test_most_sequences(checks, heads, kv, most, one_row):   # noqa: F811
    d, w = _desc(heads=heads, kv_heads=kv), heads * 64
    assert checks.desc(C.byref(d)) == 0
    x = _rows(q_stride=w, k_stride=w, v_stride=w, q_out_stride=w)
    for seqs, rc in ((most, 0), (most + 1, ILL_E_ARG), (1 << 22, ILL_E_ARG)):
        b = _batch(seqs=seqs, rows=min(seqs, (1 << 26) // heads), row0=None if one_row else P16)
        assert checks.attend(C.byref(d), C.byref(b), P16, w, P16, P16, 0, 0, 2 * P16, w, 1) == rc
        assert checks.append(C.byref(d), C.byref(b), C.byref(x), P16, P16) == rc
        if rc:
            assert b"sequences" in checks.message()
