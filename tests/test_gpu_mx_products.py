"""GPU tests of microscaled products where test_gpu_mx.py does not go: many rows of few columns, and powers far apart and blocks of NaN
among many columns (slices of the inner size, rows held in LDS).

Tolerances, per output, with u = 2^-24, h half a step of the output's type, z the sum of the products' sizes: a float32 sum of n products
that are exact there is off by at most n u z whatever its order, and the output is rounded once, h |y|. Of mxf8 rows for 16-bit outputs
each product of a group of eight neighbouring values loses less than 2^-12 of the largest of the group, which loses nothing: at
most 7 x 2^-12 z in all.
"""
from __future__ import annotations

import numpy as np
import pytest

from hip_buffers import Hip
from oracle import mx as O
from oracle import paged as V

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
LOST = 7 * 2.0 ** -12
GUARD = 0x5A


@pytest.fixture()
def hip():
    h = Hip()
    yield h
    h.close()


def _any(rng, rows, inner, fmt, low=97, high=157):
    """Rows of any codes (but NaN's) under powers far apart, as they lie in memory."""
    n = inner if fmt == "mxf8" else inner // 2
    codes = rng.integers(0, 256, (rows, n), dtype=np.uint8)
    if fmt == "mxf8":
        codes[codes & 127 == 127] = 0
    return codes, rng.integers(low, high + 1, (rows, inner // 32), dtype=np.uint8)


def _product(hip, x, w, fmt, dtype, stride=0):
    """The outputs' values; nothing is written beside them."""
    from instantllm_amd import mx
    rows, cols, inner = len(x[0]), len(w[0]), x[1].shape[1] * 32
    stride = stride or cols
    guard = np.full((rows + 1, stride), GUARD, np.uint32 if dtype == "f32" else np.uint16)
    dy = hip.put(guard)
    mx.product(*map(hip.put, (*x, *w)), dy, rows, cols, inner, format=fmt, dtype=dtype, y_stride=stride)
    got = hip.get(dy, guard)
    assert np.array_equal(got[-1], guard[-1]) and np.array_equal(got[:, cols:], guard[:, cols:]), "written outside the output"
    got = np.ascontiguousarray(got[:-1, :cols])
    return got.view(np.float32).astype(np.float64) if dtype == "f32" else V.from_bits(got, dtype)


def _check(val, x, w, fmt, dtype):
    with np.errstate(invalid="ignore"):
        xv, wv = O.values(*x, fmt), O.values(*w, "mxf4")
        y, z = xv @ wv.T, np.abs(xv) @ np.abs(wv).T
    lost = LOST if fmt == "mxf8" and dtype != "f32" else 0.0
    assert np.array_equal(np.isnan(val), np.isnan(y)), np.argwhere(np.isnan(val) != np.isnan(y))[:4]
    f = ~np.isnan(y)
    bad = np.abs(val - y)[f] > (V.HALF_STEP[dtype] * np.abs(y) + (lost + (xv.shape[1] + 1) * U) * z + V.LEAST[dtype])[f]
    assert not bad.any(), (np.argwhere(f)[bad][:4], val[f][bad][:4], y[f][bad][:4])


@pytest.mark.parametrize("fmt", ["mxf8", "mxf4"])
@pytest.mark.parametrize("rows,cols,inner", [(40000, 64, 96), (40000, 33, 160), (33000, 17, 4096), (40000, 65, 128), (30000, 128, 2080), (33000, 100, 2176), (70000, 128, 32)])
def test_many_rows_of_few_columns(hip, fmt, rows, cols, inner):
    rng = np.random.default_rng([rows, cols])
    x, w = _any(rng, rows, inner, fmt, 120, 130), _any(rng, cols, inner, "mxf4", 120, 130)
    for dtype in ("f32", "bf16"):
        print("rows", fmt, rows, cols, inner, dtype, flush=True)
        _check(_product(hip, x, w, fmt, dtype, stride=cols + 3), x, w, fmt, dtype)


# up to 16 rows from 8192 columns on are slices (one, two and four of them) or, with float32 outputs of mxf8 rows, up to 1024 values in LDS; 17 to 32 rows from
# 16384 columns on in LDS. Inner sizes whose last step has one block, two or three; numbers of steps that the slices do not divide.
MANY = [(3, 8200, 96), (16, 8200, 160), (16, 8193, 1120), (3, 8200, 1504), (5, 8197, 4000), (2, 8200, 7968), (32, 16400, 96), (17, 16387, 160), (30, 16400, 1504), (20, 16400, 992)]


@pytest.mark.parametrize("fmt", ["mxf8", "mxf4"])
@pytest.mark.parametrize("rows,cols,inner", MANY)
def test_powers_far_apart_among_many_columns(hip, fmt, rows, cols, inner):
    rng = np.random.default_rng([rows, cols, inner])
    x, w = _any(rng, rows, inner, fmt), _any(rng, cols, inner, "mxf4")
    for dtype in ("f32", "bf16"):
        print("powers", fmt, rows, cols, inner, dtype, flush=True)
        _check(_product(hip, x, w, fmt, dtype), x, w, fmt, dtype)


@pytest.mark.parametrize("fmt", ["mxf8", "mxf4"])
@pytest.mark.parametrize("rows,cols,inner", MANY)
def test_nan_blocks_among_many_columns(hip, fmt, rows, cols, inner):
    """Blocks of NaN reach their column's or row's outputs and no other: in a column's last block, where the next bytes are the next column's,
    in a column's first, in the last block of all, in one of the first step and one of the last; and in a row's first and last."""
    rng = np.random.default_rng([rows, cols, inner, 1])
    x, w = _any(rng, rows, inner, fmt, 120, 130), _any(rng, cols, inner, "mxf4", 120, 130)
    last = inner // 32 - 1
    at = [(7, last), (19, 0), (33, last), (34, 0), (4097, last // 2), (cols - 20, max(last - 1, 0)), (cols - 3, 0), (cols - 1, last)]
    for c, b in at:
        w[1][c, b] = 255
    for dtype in ("f32", "bf16"):
        print("nan columns", fmt, rows, cols, inner, dtype, flush=True)
        val = _product(hip, x, w, fmt, dtype)
        assert np.isnan(val).sum() == rows * len(at)
        _check(val, x, w, fmt, dtype)
    for r, b in ((0, last), (rows - 1, 0)):
        x[1][r, b] = 255
    for dtype in ("f32", "bf16"):
        print("nan rows", fmt, rows, cols, inner, dtype, flush=True)
        val = _product(hip, x, w, fmt, dtype)
        assert np.isnan(val).sum() == rows * len(at) + 2 * (cols - len(at))
        _check(val, x, w, fmt, dtype)
