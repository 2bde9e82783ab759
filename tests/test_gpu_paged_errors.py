"""GPU test: an error of the program's own HIP calls, not yet fetched, is not taken for the paged-cache operators'."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from hip_buffers import Hip
from test_gpu_paged import Setup

pytestmark = pytest.mark.gpu


@pytest.fixture()
def hip():
    h = Hip()
    yield h
    h.close()


@pytest.mark.parametrize("seqs,heads,kv", [([(300, 1)], 4, 2), ([(150, 150)], 112, 112), ([(150, 150), (9, 1)], 112, 112)], ids=["step", "prompt", "both"])
def test_an_earlier_error_of_the_program(hip, seqs, heads, kv):
    s = Setup(hip, seqs, heads=heads, kv=kv)
    w = heads * 64
    q = s.random_bits(s.rows, w)
    want = s.attend(q=q)
    dq, do, dk = hip.put(q), hip.put(np.zeros_like(want)), hip.put(s.random_bits(s.rows, (heads + 2 * kv) * 64))
    bad = lambda: hip.h.hipMemcpy(None, C.c_void_p(s.kc), 16, 99)   # noqa: E731  (no such kind of copy: refused on the host)
    assert bad() != 0
    s.op.attend(s.batch, s.kc, s.vc, dq, do)
    assert np.array_equal(hip.get(do, want), want)
    assert bad() != 0
    s.op.append(s.batch, s.kc, s.vc, k=dk, v=dk + 2 * kv * 64, x_stride=(heads + 2 * kv) * 64)
    hip.sync()
    assert hip.h.hipGetLastError() != 0   # the program's, still there
    assert hip.h.hipGetLastError() == 0
