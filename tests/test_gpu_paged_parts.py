"""GPU tests of the paged-cache attention where a prompt's keys are cut into more than 16 parts, which are joined in two steps
(test_paged_parts.py counts the parts on the CPU). Tolerances: test_gpu_paged.py."""
from __future__ import annotations

import numpy as np
import pytest

from hip_buffers import Hip
from test_gpu_paged import Setup

pytestmark = pytest.mark.gpu

# (sequences, query heads, key/value heads, parts that the first sequence's keys are cut into): a long sequence beside many short
# ones, so that the prompt kernel runs and the long one is far over the average share
SHAPES = [([(9000, 16)] + [(40, 40)] * 110, 8, 1, 36), ([(9000, 40)] + [(40 + i % 3, 40) for i in range(230)], 4, 1, 24)]


@pytest.fixture()
def hip():
    h = Hip()
    yield h
    h.close()


@pytest.mark.parametrize("dim,dtype", [(64, "f16"), (128, "bf16")])
@pytest.mark.parametrize("seqs,heads,kv,parts", SHAPES, ids=[str(s[3]) for s in SHAPES])
def test_prompts_joined_in_two_steps(hip, seqs, heads, kv, parts, dim, dtype):
    s = Setup(hip, seqs, heads=heads, kv=kv, dim=dim, dtype=dtype)
    q = s.random_bits(s.rows, heads * dim)
    first = s.attend(q=q)
    s.attend(q=q, out_dtype="f32")
    s.attend(q=q, window=8000, sinks=70)
    for _ in range(3):   # the same bits, whichever part ends last
        assert np.array_equal(s.attend(q=q, check=False), first)
