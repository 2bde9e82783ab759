"""GPU tests of what the sums of mxf8 rows' products for 16-bit outputs are off by, as include/ill_hip.h states it: of eight neighbouring
values' products each loses less than 2^-12 of the largest one's size, and the largest nothing.

Outputs are rounded to 16 bits, which hides that. What cancels shows it: a product next to a large one that another group takes back, or a
sum and a bias that is minus its value. Then, with u = 2^-24 and z the sum of the products' sizes, an output may be off by 7 x 2^-12 of the sum
of the groups' largest products, by (n + 2) u z for n float32 additions and the bias's own rounding, and by half a step of what is left.
"""
from __future__ import annotations

import numpy as np
import pytest

from hip_buffers import Hip
from oracle import mx as O
from oracle import paged as V

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture()
def hip():
    h = Hip()
    yield h
    h.close()


def _product(hip, x, w, bias=None):
    from instantllm_amd import mx
    rows, cols, inner = len(x[0]), len(w[0]), x[1].shape[1] * 32
    like = np.empty((rows, cols), np.uint16)
    dy = hip.alloc(like.nbytes)
    mx.product(*map(hip.put, (*x, *w)), dy, rows, cols, inner, format="mxf8", dtype="bf16", bias=None if bias is None else hip.put(bias))
    return V.from_bits(hip.get(dy, like), "bf16")


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("at", [1, 7])
def test_every_small_product_beside_every_large_one(hip, sign, at):
    """One group: a large product and a small one; the next group: minus the large one. What is left has six bits at most, and is
    exact in bf16."""
    a, b = (v.ravel() for v in np.meshgrid(np.arange(1, 127), np.arange(1, 127), indexing="ij"))
    u, v = (v.ravel() for v in np.meshgrid(np.arange(1, 8), np.arange(1, 8), indexing="ij"))
    x, w = np.zeros((len(a), 32), np.uint8), np.zeros((len(u), 32), np.uint8)
    x[:, 0], x[:, at], x[:, 8] = a, b + (128 if sign < 0 else 0), a
    w[:, 0], w[:, at], w[:, 8] = u, v, u | 8
    one = lambda n: np.full((n, 1), 127, np.uint8)
    wt = (O.pack(w, "mxf4"), one(len(u)))
    large = np.outer(O.E4M3[a], O.E2M1[u])
    small = sign * np.outer(O.E4M3[b], O.E2M1[v])
    lower = np.minimum(large, np.abs(small))
    for rows in (slice(None), slice(5000, 5016)):   # tiles, and up to 16 rows
        got = _product(hip, (x[rows], one(len(a[rows]))), wt)
        assert (np.abs(got - small[rows]) < 2.0 ** -12 * np.maximum(large, np.abs(small))[rows]).all()
        exact = (lower >= 2.0 ** -6 * np.maximum(large, np.abs(small)))[rows]   # (six bits of each, above 2^-12 of the larger one)
        assert np.array_equal(got[exact], small[rows][exact])


def _values(kind, rng, cols, inner):
    if kind == "spread":   # codes, and powers, of evenly spread exponents
        x = rng.integers(0, 127, (1, inner), dtype=np.uint8) + 128 * rng.integers(0, 2, (1, inner), dtype=np.uint8)
        power = lambda rows: rng.integers(110, 130, (rows, inner // 32), dtype=np.uint8)
        return (x.astype(np.uint8), power(1)), (rng.integers(0, 256, (cols, inner // 2), dtype=np.uint8), power(cols))
    x = rng.standard_normal((1, inner))
    if kind == "outliers":
        x[:, ::61] *= 50
    return O.quantize(x, "mxf8"), O.quantize(rng.standard_normal((cols, inner)), "mxf4")


@pytest.mark.parametrize("kind", ["normal", "outliers", "spread"])
@pytest.mark.parametrize("rows,cols,inner", [(1, 2000, 96), (1, 2000, 4864), (16, 8200, 896), (3, 8200, 2080), (20, 16400, 128), (200, 2000, 896), (600, 2000, 928)])
def test_sums(hip, kind, rows, cols, inner):
    """The same row `rows` times, and a bias of minus its result."""
    rng = np.random.default_rng([cols, inner])
    x, w = _values(kind, rng, cols, inner)
    xv, wv = O.values(*x, "mxf8"), O.values(*w, "mxf4")
    p = wv * xv
    y, z = p.sum(1), np.abs(p).sum(1)
    largest = np.abs(p).reshape(cols, -1, 8).max(2).sum(1)
    bias = (-y).astype(np.float32)
    left = y + bias.astype(np.float64)
    got = _product(hip, tuple(np.repeat(a, rows, 0) for a in x), w, bias)
    assert (got == got[:1]).all()
    off = got[0] - left
    assert (np.abs(off) <= 7 * 2.0 ** -12 * largest + (inner + 2) * U * z + V.HALF_STEP["bf16"] * np.abs(got[0])).all()
    # Normal values, by the 2-norm. A block's largest code is 256 to 448, 2.1 standard deviations (of 32 values): s is 120 at least, and 2 of w's 6. The largest
    # product there is, 2688, makes the others lose less than 2^-2 each (2^11 x 2^-13), and only those of sizes below 4 of x, whose bits lie lower: 3 of 100
    # values. sqrt(0.03 / 3) x 2^-2 / (120 x 2) = 1.1e-4.
    if kind == "normal":
        assert np.linalg.norm(off) <= 1.1e-4 * np.linalg.norm(y)
    print("sums", kind, rows, cols, inner, np.linalg.norm(off) / np.linalg.norm(y), (np.abs(off) / z).max(), flush=True)
