"""GPU tests of the paged-cache attention with bf16 values near the ends of float32's range, against the float64 restatement by
the tolerances of test_gpu_paged.py. Sums are of weights of at most 1: they stay below 2^128 where the number of keys times the
greatest value does. (N normal values are below 6 here: 9000 x 6 < 2^16, 1000 x 6 < 2^13.)"""
from __future__ import annotations

import numpy as np
import pytest

from hip_buffers import Hip
from oracle import paged as O
from test_gpu_paged import Setup

pytestmark = pytest.mark.gpu


@pytest.fixture()
def hip():
    h = Hip()
    yield h
    h.close()


@pytest.mark.parametrize("out_dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("power", [2.0 ** 112, 2.0 ** -90], ids=["large", "small"])
@pytest.mark.parametrize("seqs,heads,kv", [([(1000, 1), (300, 1), (3, 1)], 4, 2), ([(1000, 150), (300, 128)], 112, 112), ([(9000, 20)], 4, 1)],
                         ids=["step", "prompt-kernel", "parts"])
def test_bf16_values_near_the_ends_of_the_range(hip, seqs, heads, kv, power, dim, out_dtype):
    """Even scores and steep ones; values of one sign in every second dim, so that their sums grow with the keys."""
    s = Setup(hip, seqs, heads=heads, kv=kv, dim=dim, dtype="bf16")
    v = s.rng.standard_normal((s.pages, s.page, kv, dim), dtype=np.float32)
    assert np.abs(v).max() < 6
    v[..., ::2] = np.abs(v[..., ::2])
    s.view(s.v_bits)[...] = O.to_bits(v * np.float32(power), "bf16")
    for steep in (0.02, 2.0):
        q = s.rng.standard_normal((s.rows, heads * dim), dtype=np.float32) * np.float32(steep)
        s.attend(q=O.to_bits(q, "bf16"), out_dtype=out_dtype)
        s.attend(q=O.to_bits(q, "bf16"), out_dtype=out_dtype, window=200, sinks=3)
