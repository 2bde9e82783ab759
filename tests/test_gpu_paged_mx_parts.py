"""GPU tests of attention over microscaled caches where keys are cut into more than 16 parts, which are joined in two steps in LDS that held
the tiles (test_paged_parts.py counts the prompts' parts on the CPU), and of batches on either side of 256 sequences, up to which the units
of many keys are launched first. Tolerances: test_gpu_paged_mx.py."""
from __future__ import annotations

import numpy as np
import pytest

from hip_buffers import Hip
from test_gpu_paged_mx import MxSetup
from test_gpu_paged_parts import SHAPES

pytestmark = pytest.mark.gpu


@pytest.fixture()
def hip():
    h = Hip()
    yield h
    h.close()


def _attend(s, **call):
    q = s.random_bits(s.rows, s.heads * s.dim)
    first = s.attend(q=q, **call)
    s.attend(q=q, out_dtype="f32", **call)
    for _ in range(3):   # the same bits, whichever part ends last
        assert np.array_equal(s.attend(q=q, check=False, **call), first)


@pytest.mark.parametrize("dim,dtype", [(64, "f16"), (128, "bf16")])
@pytest.mark.parametrize("seqs,heads,kv,parts", SHAPES, ids=[str(s[3]) for s in SHAPES])
def test_prompts_joined_in_two_steps(hip, seqs, heads, kv, parts, dim, dtype):
    _attend(MxSetup(hip, seqs, heads=heads, kv=kv, dim=dim, dtype=dtype))


@pytest.mark.parametrize("dim,dtype", [(64, "bf16"), (128, "f16")])
@pytest.mark.parametrize("rows", [1, 3, 16])   # of the long sequence: joined by four, two (heads of 64) or one group of threads
def test_steps_joined_in_two_steps(hip, rows, dim, dtype):
    _attend(MxSetup(hip, [(20000, rows), (17, 1)], heads=2, kv=1, dim=dim, dtype=dtype))


@pytest.mark.parametrize("dim,dtype", [(64, "f16"), (128, "bf16")])
@pytest.mark.parametrize("seqs", [256, 257, 300])
def test_many_sequences(hip, seqs, dim, dtype):
    rng = np.random.default_rng(seqs)
    lens = [(int(n), 1) for n in np.exp(rng.uniform(0, np.log(1500), seqs))]
    lens[seqs // 2] = (6000, 1)
    _attend(MxSetup(hip, lens, heads=4, kv=2, dim=dim, dtype=dtype, one_row=True))
    lens[3], lens[seqs - 2] = (400, 90), (700, 33)
    _attend(MxSetup(hip, lens, heads=4, kv=2, dim=dim, dtype=dtype), window=300, sinks=20)
