"""GPU tests of the microscaled operators (instantllm_amd.mx over the C ABI) against their float64 restatement (oracle/mx.py).

Quantisation is exact: its inputs' values, a division by a power of two and one rounding; codes and powers have to be the
restatement's, bit for bit. Values that come back are rounded once, where the type has no place for them.

Tolerances of products, per output, with u = 2^-24, h half a step of the output's type, z the sum of the products' sizes (the
bias's among them): products of codes and powers are exact in float32. A sum of n of them in float32 is off by at most n u z whatever
its order; the output is rounded once, h |y|. Of mxf8 rows for 16-bit outputs the matrix units drop parts of a group's products: what the
header allows for that is half a step of f16 of z, 2^-11 z. All values of a normal product together (the 2-norm) are off by
less than h in 16 bits, whose rounding alone is h / sqrt 3, and less than 1e-6 in float32.
"""
from __future__ import annotations

import numpy as np
import pytest

from hip_buffers import Hip
from oracle import mx as O
from oracle import paged as V

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
GUARD = 0x5A


@pytest.fixture()
def hip():
    h = Hip()
    yield h
    h.close()


def _bits(x, dtype):
    """(array as it lies in memory, its values)."""
    b = V.to_bits(x, dtype)
    return b, V.from_bits(b, dtype)


def _spread(rng, rows, cols):
    x = rng.standard_normal((rows, cols), dtype=np.float32) * np.exp(rng.standard_normal((rows, 1), dtype=np.float32))
    x[:, ::61] *= 8
    return x


def _quantize(hip, bits, fmt, dtype, cols, stream=None):
    """What the call writes, with guards behind both arrays."""
    from instantllm_amd import mx
    rows, stride = bits.shape
    codes = np.full(rows * mx.code_bytes(fmt, cols) + 64, GUARD, np.uint8)
    powers = np.full(rows * cols // 32 + 64, GUARD, np.uint8)
    dx, dc, dp = hip.put(bits), hip.put(codes), hip.put(powers)
    mx.quantize(dx, dc, dp, rows, cols, format=fmt, dtype=dtype, x_stride=stride, stream=stream)
    codes, powers = hip.get(dc, codes), hip.get(dp, powers)
    assert (codes[-64:] == GUARD).all() and (powers[-64:] == GUARD).all(), "written behind the rows"
    return codes[:-64].reshape(rows, -1), powers[:-64].reshape(rows, -1), dc, dp


@pytest.mark.parametrize("fmt", ["mxf8", "mxf4"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols,extra", [(1, 32, 0), (1, 896, 0), (3, 96, 8), (257, 4864, 16), (70, 160, 0), (1, 32 * 1031, 0)])
def test_quantize_matches_oracle(hip, fmt, dtype, rows, cols, extra):
    print("quantize", fmt, dtype, rows, cols, extra, flush=True)
    rng = np.random.default_rng([rows, cols])
    bits, x = _bits(_spread(rng, rows, cols + extra), dtype)
    codes, powers, _, _ = _quantize(hip, bits, fmt, dtype, cols)
    want = O.quantize(x[:, :cols], fmt)
    assert np.array_equal(powers, want[1]) and np.array_equal(codes, want[0])


@pytest.mark.parametrize("fmt", ["mxf8", "mxf4"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_quantize_borders(hip, fmt, dtype):
    """Every code and every border between two, next to the largest sizes a block may have; the ends of the type's range; blocks
    of zeros, and ones that hold an infinity or NaN."""
    sizes = O.SIZES[fmt]
    at = np.concatenate([sizes, (sizes[1:] + sizes[:-1]) / 2])
    blocks = []
    for power in (-20, -3, 0, 5):
        for most in (sizes[-1], 2.0 ** O.TOP[fmt], 2.0 ** O.TOP[fmt] * 1.99):
            for s in range(0, len(at), 31):
                b = np.zeros(32)
                b[0] = most
                part = at[s:s + 31]
                b[1:1 + len(part)] = np.minimum(part, most) * (-1) ** np.arange(len(part))
                blocks.append(b * 2.0 ** power)
    least = V.LEAST[dtype]
    most = {"f32": 3.4e38, "f16": 65504.0, "bf16": 3.38e38}[dtype]
    for v in (0.0, -0.0, least, 3 * least, most, -most, np.inf, -np.inf, np.nan):
        b = np.zeros(32)
        b[5], b[6] = v, 1.0 if not np.isfinite(v) else 0.0
        blocks.append(b)
        blocks.append(np.full(32, v))
    with np.errstate(over="ignore"):
        bits, x = _bits(np.array(blocks).astype(np.float32).reshape(1, -1), dtype)
    codes, powers, dc, dp = _quantize(hip, bits, fmt, dtype, x.shape[1])
    want = O.quantize(x, fmt)
    assert np.array_equal(powers, want[1]) and np.array_equal(codes, want[0])
    _back(hip, dc, dp, want[0], want[1], fmt, "f32")


def _back(hip, dc, dp, codes, powers, fmt, dtype, extra=0):
    from instantllm_amd import mx
    rows, cols = codes.shape[0], powers.shape[1] * 32
    guard = np.full((rows, cols + extra), GUARD, np.uint32 if dtype == "f32" else np.uint16)
    dy = hip.put(guard)
    mx.dequantize(dc, dp, dy, rows, cols, format=fmt, dtype=dtype, y_stride=cols + extra)
    got = hip.get(dy, guard)
    assert np.array_equal(got[:, cols:], guard[:, cols:]), "written between the rows"
    y = O.values(codes, powers, fmt)
    with np.errstate(over="ignore"):
        want = V.from_bits(V.to_bits(y.astype(np.float32), dtype), dtype) if dtype != "f32" else y.astype(np.float32).astype(np.float64)
    val = V.from_bits(np.ascontiguousarray(got[:, :cols]), dtype) if dtype != "f32" else np.ascontiguousarray(got[:, :cols]).view(np.float32).astype(np.float64)
    assert np.array_equal(val, want, equal_nan=True), np.argwhere(~((val == want) | (np.isnan(val) & np.isnan(want))))[:4]


@pytest.mark.parametrize("fmt", ["mxf8", "mxf4"])
@pytest.mark.parametrize("dtype,extra", [("f32", 0), ("f16", 8), ("bf16", 0), ("f32", 4)])
def test_dequantize_every_code_and_power(hip, fmt, dtype, extra):
    """All codes under all powers; the types' ends are rounded to as elsewhere (powers next to 2^127 leave every type's range)."""
    n = 256 if fmt == "mxf8" else 32
    codes = np.arange(256, dtype=np.uint8) if fmt == "mxf8" else O.pack(np.arange(32, dtype=np.uint8) & 15, fmt)
    codes = np.repeat(codes.reshape(1, -1), 256, 0)
    powers = np.repeat(np.arange(256, dtype=np.uint8).reshape(-1, 1), n // 32, 1)
    _back(hip, hip.put(codes), hip.put(powers), codes, powers, fmt, dtype, extra)


# ---- products ------------------------------------------------------------------------------
class Product:
    """Rows, a matrix and a bias on the device, and their values."""

    def __init__(self, hip, rows, cols, inner, fmt, seed=0, bias=False, x=None, w=None):
        self.hip, self.rows, self.cols, self.inner, self.fmt = hip, rows, cols, inner, fmt
        rng = self.rng = np.random.default_rng([seed, rows, cols, inner])
        self.held = O.quantize(_spread(rng, rows, inner) if x is None else x, fmt)
        if w is None and cols * inner > 1 << 21:   # (quicker: any codes)
            self.w = (rng.integers(0, 256, (cols, inner // 2), dtype=np.uint8), rng.integers(116, 122, (cols, inner // 32), dtype=np.uint8))
        else:
            self.w = O.quantize(rng.standard_normal((cols, inner), dtype=np.float32) * 0.05 if w is None else w, "mxf4")
        self.bias = rng.standard_normal(cols, dtype=np.float32) if bias else None
        self.dev = [hip.put(a) for a in (*self.held, *self.w)]
        self.d_bias = hip.put(self.bias) if bias else None

    def sums(self):
        x, w = O.values(*self.held, self.fmt), O.values(*self.w, "mxf4")
        y, z = x @ w.T, np.abs(x) @ np.abs(w).T
        return (y, z) if self.bias is None else (y + self.bias, z + np.abs(self.bias))

    def run(self, dtype, extra=0, stream=None):
        from instantllm_amd import mx
        guard = np.full((self.rows + 1, self.cols + extra), GUARD, np.uint32 if dtype == "f32" else np.uint16)
        dy = self.hip.put(guard)
        mx.product(*self.dev, dy, self.rows, self.cols, self.inner, format=self.fmt, dtype=dtype, bias=self.d_bias, y_stride=self.cols + extra, stream=stream)
        got = self.hip.get(dy, guard)
        assert np.array_equal(got[-1], guard[-1]) and np.array_equal(got[:, self.cols:], guard[:, self.cols:]), "written outside the output"
        return np.ascontiguousarray(got[:-1, :self.cols])

    def check(self, got, dtype, norm=True):
        y, z = self.sums()
        val = V.from_bits(got, dtype) if dtype != "f32" else got.view(np.float32).astype(np.float64)
        h = V.HALF_STEP[dtype]
        cut = 2.0 ** -11 if self.fmt == "mxf8" and dtype != "f32" else 0.0
        bad = ~(np.abs(val - y) <= h * np.abs(y) + (cut + (self.inner + 1) * U) * z + V.LEAST[dtype])
        assert not bad.any(), (np.argwhere(bad)[:4], val[bad][:4], y[bad][:4])
        if norm:
            assert np.linalg.norm(val - y) <= (1e-6 if dtype == "f32" else h) * np.linalg.norm(y)


SHAPES = [   # rows, columns, inner size: single rows, batches, prompts; odd sizes; inner sizes that are no multiple of 128
    (1, 1152, 896), (1, 896, 4864), (1, 1, 32), (2, 17, 64), (7, 33, 96), (16, 100, 160), (16, 20001, 256), (17, 1152, 896), (31, 48, 4864), (33, 70, 288),
    (64, 130, 896), (65, 128, 128), (100, 257, 512), (128, 129, 384), (200, 1000, 2048), (333, 515, 1152), (513, 300, 4864), (1, 17000, 32), (40, 16500, 96), (1025, 1030, 256),
    # inner sizes that are no multiple of 128, in tiles: one to three blocks more, one stage and several, one or two columns, the last row alone
    (17, 1, 32), (18, 3, 96), (65, 2, 64), (129, 200, 32), (64, 65, 160), (193, 130, 1120), (70, 4200, 672), (1100, 2100, 416), (1100, 2100, 1056), (257, 8200, 64),
    # many columns: slices of the inner size, one to eight, and rows held in LDS
    (5, 8200, 1504), (16, 8192, 4000), (3, 8300, 8192), (20, 16500, 896), (32, 17000, 96), (1, 8193, 8320),
    # tiles of every size, of four and eight waves: 128 x 128, 128 x 64, 128 x 128 and 256 x 128 (mxf8), 128 x 128 twice, 128 x 256 and 256 x 256 (mxf4)
    (1900, 2000, 128), (2200, 2300, 384), (3001, 2450, 256), (6450, 3850, 128), (4001, 4002, 4096),
    (1900, 2000, 224), (2200, 2300, 352), (2200, 2300, 64), (6450, 3850, 160), (6450, 3850, 96), (4001, 4002, 4064), (4001, 4002, 4128)]


@pytest.mark.parametrize("fmt", ["mxf8", "mxf4"])
@pytest.mark.parametrize("rows,cols,inner", SHAPES)
def test_product_matches_oracle(hip, fmt, rows, cols, inner):
    p = Product(hip, rows, cols, inner, fmt, bias=(rows + cols) % 2 == 0)
    for dtype in ("f32", "f16", "bf16"):
        print("product", fmt, rows, cols, inner, dtype, flush=True)
        p.check(p.run(dtype, extra=(rows % 3) * 3), dtype)


@pytest.mark.parametrize("rows", [3, 70, 300])
def test_product_of_extreme_powers(hip, rows):
    """Powers far apart in a row, zeros, and codes of evenly spread exponents."""
    rng = np.random.default_rng(rows)
    x = rng.standard_normal((rows, 256)) * 2.0 ** rng.integers(-30, 5, (rows, 256))
    x[:, :32] *= 2.0 ** -60
    x[0] = 0
    w = rng.standard_normal((150, 256)) * np.repeat(2.0 ** rng.integers(-40, 10, (150, 8)), 32, 1)
    for fmt in ("mxf8", "mxf4"):
        p = Product(hip, rows, 150, 256, fmt, x=x, w=w)
        for dtype in ("f32", "bf16"):
            print(fmt, dtype, flush=True)
            p.check(p.run(dtype), dtype, norm=False)


@pytest.mark.parametrize("fmt", ["mxf8", "mxf4"])
@pytest.mark.parametrize("rows,inner", [(2, 96), (40, 256), (200, 256), (30, 160), (200, 224)])
def test_product_of_nan_blocks(hip, fmt, rows, inner):
    """A NaN block reaches the outputs of its row or column, and no other."""
    rng = np.random.default_rng(5)
    x, w = rng.standard_normal((rows, inner)), rng.standard_normal((140, inner))
    x[1, inner - 1] = np.nan
    w[17, 3] = np.inf
    p = Product(hip, rows, 140, inner, fmt, x=x, w=w)
    y, _ = p.sums()
    for dtype in ("f32", "f16"):
        got = p.run(dtype)
        val = V.from_bits(got, dtype) if dtype != "f32" else got.view(np.float32).astype(np.float64)
        assert np.array_equal(np.isnan(val), np.isnan(y)) and np.isnan(y).sum() == 140 + rows - 1


def test_no_rows(hip):
    from instantllm_amd import mx
    guard = np.full(64, GUARD, np.uint8)
    d = hip.put(guard)
    mx.quantize(d, d, d, 0, 32)
    mx.dequantize(d, d, d, 0, 32)
    mx.product(d, d, d, d, d, 0, 16, 32)
    assert np.array_equal(hip.get(d, guard), guard)


def test_streams_and_graphs(hip):
    """A layer's two calls captured and replayed while its input changes, beside eager calls on another stream."""
    from instantllm_amd import mx
    rng = np.random.default_rng(3)
    rows, cols, inner = 20, 300, 512
    w = O.quantize(rng.standard_normal((cols, inner)), "mxf4")
    dw = [hip.put(a) for a in w]
    out = np.empty((rows, cols), np.float32)
    bufs = [(hip.alloc(rows * inner * 2), hip.alloc(rows * inner), hip.alloc(rows * inner // 32), hip.alloc(out.nbytes)) for _ in range(2)]

    def work(b, stream):
        mx.quantize(b[0], b[1], b[2], rows, inner, dtype="bf16", stream=stream)
        mx.product(b[1], b[2], *dw, b[3], rows, cols, inner, dtype="f32", stream=stream)
    s1, s2 = hip.stream(), hip.stream()
    graph = hip.capture(s1, lambda: work(bufs[0], s1))
    for _ in range(4):
        xs = [V.to_bits(_spread(rng, rows, inner), "bf16") for _ in bufs]
        for b, x in zip(bufs, xs):
            hip.write(b[0], x)
        hip.launch(graph, s1)
        work(bufs[1], s2)
        hip.sync()
        for b, x in zip(bufs, xs):
            q = O.values(*O.quantize(V.from_bits(x, "bf16"), "mxf8"), "mxf8")
            wv = O.values(*w, "mxf4")
            assert (np.abs(hip.get(b[3], out) - q @ wv.T) <= (inner + 2) * U * (np.abs(q) @ np.abs(wv).T)).all()


@pytest.mark.parametrize("fmt", ["mxf8", "mxf4"])
@pytest.mark.parametrize("rows,cols,inner", [(3, 40, 96), (5, 8200, 256), (20, 16400, 128), (70, 200, 128), (70, 200, 160)])
def test_outputs_aligned_to_their_type(hip, fmt, rows, cols, inner):
    """Outputs from any element on: the same values as from an aligned one, and none beside them."""
    from instantllm_amd import mx
    p = Product(hip, rows, cols, inner, fmt)
    for dtype in ("f32", "bf16"):
        size = 4 if dtype == "f32" else 2
        want = p.run(dtype)
        for off in (1, 4):
            print("offset", fmt, rows, cols, inner, dtype, off, flush=True)
            guard = np.full(rows * cols + off + 1, GUARD, want.dtype)
            dy = hip.put(guard)
            mx.product(*p.dev, dy + size * off, rows, cols, inner, format=fmt, dtype=dtype)
            got = hip.get(dy, guard)
            assert np.array_equal(got[off:-1], want.ravel()) and (got[:off] == GUARD).all() and got[-1] == GUARD


def test_rows_past_32_bits(hip):
    """More than 2^32 values, and rows more than 2^32 bytes apart."""
    from instantllm_amd import mx
    rng = np.random.default_rng(8)
    rows, cols, few = (1 << 16) + 3, 1 << 16, 3
    bits, x = _bits(_spread(rng, few, cols), "bf16")
    dx, dc, dp = hip.alloc(2 * rows * cols), hip.alloc(rows * cols), hip.alloc(rows * cols // 32)
    hip.write(dx + 2 * (rows - few) * cols, bits)
    for fmt in ("mxf8", "mxf4"):
        print("rows", fmt, flush=True)
        mx.quantize(dx, dc, dp, rows, cols, format=fmt, dtype="bf16")
        want = O.quantize(x, fmt)
        assert np.array_equal(hip.get(dc + mx.code_bytes(fmt, (rows - few) * cols), want[0]), want[0])
        assert np.array_equal(hip.get(dp + (rows - few) * cols // 32, want[1]), want[1])
    stride = (1 << 31) + 8
    held = O.quantize(x[:2], "mxf8")
    hip.write(dc, held[0])
    hip.write(dp, held[1])
    mx.dequantize(dc, dp, dx, 2, cols, dtype="bf16", y_stride=stride)
    back = O.values(*held, "mxf8")
    for r in range(2):
        assert np.array_equal(V.from_bits(hip.get(dx + 2 * r * stride, bits[0]), "bf16"), back[r])
    other = [hip.alloc(held[0].nbytes), hip.alloc(held[1].nbytes)]
    mx.quantize(dx, *other, 2, cols, dtype="bf16", x_stride=stride)
    assert np.array_equal(O.values(hip.get(other[0], held[0]), hip.get(other[1], held[1]), "mxf8"), back)
    w = O.quantize(rng.standard_normal((24, 256), dtype=np.float32), "mxf4")
    dw = [hip.put(a) for a in w]
    two = O.quantize(x[:2, :256], "mxf8")
    near = hip.alloc(2 * 24 * 2)
    d2 = [hip.put(a) for a in two]
    mx.product(*d2, *dw, near, 2, 24, 256, dtype="bf16")
    mx.product(*d2, *dw, dx, 2, 24, 256, dtype="bf16", y_stride=stride)
    want = hip.get(near, np.empty((2, 24), np.uint16))
    for r in range(2):
        assert np.array_equal(hip.get(dx + 2 * r * stride, want[r]), want[r])


@pytest.mark.parametrize("fmt", ["mxf8", "mxf4"])
def test_operands_past_32_bits(hip, fmt):
    """The last columns of a matrix, and the last rows, whose codes are more than 2^32 bytes: as in a product of those alone."""
    from instantllm_amd import mx
    rng = np.random.default_rng(9)
    last, inner, cols = 40, 8192, (1 << 20) + 40
    w = (rng.integers(0, 256, (last, inner // 2), dtype=np.uint8), rng.integers(116, 122, (last, inner // 32), dtype=np.uint8))
    big = [hip.alloc(cols * inner // 2), hip.alloc(cols * inner // 32)]   # (what the others hold reaches their outputs only)
    for d, a in zip(big, w):
        hip.write(d + (cols - last) * a.shape[1], a)
    for rows in (3, 40, 300):
        p = Product(hip, rows, last, inner, fmt, w=np.zeros((last, inner), np.float32))
        p.w = w
        dy = hip.alloc(rows * cols * 2)
        print("columns", fmt, rows, flush=True)
        mx.product(*p.dev[:2], *big, dy, rows, cols, inner, format=fmt, dtype="f16")
        got = np.stack([hip.get(dy + 2 * (r * cols + cols - last), np.empty(last, np.uint16)) for r in range(rows)])
        p.check(got, "f16", norm=False)
    for inner in (16384, 16384 + 32):
        rows, cols, last = (1 << 19) + 70, 70, 70
        p = Product(hip, last, cols, inner, fmt)
        big = [hip.alloc(rows * a.shape[1]) for a in p.held]
        for d, a in zip(big, p.held):
            hip.write(d + (rows - last) * a.shape[1], a)
        dy = hip.alloc(rows * cols * 4)
        for dtype in ("f16", "f32"):
            print("rows", fmt, inner, dtype, flush=True)
            mx.product(*big, *p.dev[2:], dy, rows, cols, inner, format=fmt, dtype=dtype)
            size = 4 if dtype == "f32" else 2
            p.check(hip.get(dy + size * (rows - last) * cols, np.empty((last, cols), np.uint32 if size == 4 else np.uint16)), dtype, norm=False)
