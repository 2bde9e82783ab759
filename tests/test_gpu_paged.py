"""GPU tests of the paged-cache operators (PagedAttention over the C ABI) against their float64 restatement (oracle/paged.py).

Tolerances, per value, with u = 2^-24 (half a step of float32 relative to the value) and h half a step of the output's type:
append: the result is rounded once, h |y|, from float32 arithmetic on values of size z (the sum of the sizes of the pair that the
  rotation mixes): bias 1 u; mean of squares, square root and two products of the norm: (16 + 3 + 7) / 2 + 4 < 18 u; sine and cosine: the
  turn's rounding 2^-26, times 2 pi, < 2 u, and two units in the last place, 4 u; two products and a sum 3 u; the two sides' angles in float64
  at 2^30 positions 3 u. Together below 32 u z. Below the least normal number half a step is half of the smallest subnormal.
attend: scores are sums of D products in float32, off by at most D u times d, the greatest sum of |q k| scale; scale, the change to
  powers of 2 and the exponential add at most 8 u d + 2^-21. A softmax weight is off by at most twice that relative to itself, and sums of N
  weights and values by N u each. Weights are rounded for the product with the values to the cache's type (for float32
  outputs in parts: two of f16 2^-22, three of bf16 2^-24). All of these are relative to z, the weighted sum of the values' sizes. The output is rounded once, h |y|.
These are bounds; the errors are nearly independent, so all values together are off by less than 1.5 h (the output's and the weights'
  rounding, uniform, are h / sqrt 3 each), and in float32 by less than 1e-5.
"""
from __future__ import annotations

import math

import numpy as np
import pytest

from hip_buffers import Hip
from oracle import paged as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
GUARD = 0x5A5A


@pytest.fixture()
def hip():
    h = Hip()
    yield h
    h.close()


class Setup:
    """A cache, a batch and its handle. seqs: (length, new rows) each. layout: axes of the cache from the outermost in, 'p' pages, 's'
    slots, 'h' heads; a digit widens the stride of the axis before it by so many times 8."""

    def __init__(self, hip, seqs, heads=14, kv=2, dim=64, dtype="f16", page=16, layout="psh", one_row=False, pad=0, seed=0, spare=3, max_rows=0,
                 shuffle=True, **kw):
        from instantllm_amd.paged import PagedAttention
        self.hip, self.rng = hip, np.random.default_rng([seed, heads, dim, page])
        self.heads, self.kv, self.dim, self.dtype, self.page = heads, kv, dim, dtype, page
        self.lens = np.array([n for n, _ in seqs], np.int32)
        counts = [c for _, c in seqs]
        self.row0 = None if one_row else np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.total = sum(counts)
        self.rows = self.total + pad
        need = [-(-max(n, 0) // page) for n, _ in seqs]
        self.pages = sum(need) + spare
        order = self.rng.permutation(self.pages) if shuffle else np.arange(self.pages)
        self.width = max(need + [1])
        self.table = np.full((len(seqs), self.width + 2), 1 << 30, np.int32)   # entries behind the last are not read
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        extent, strides, step = {"p": self.pages, "s": page, "h": kv}, {}, dim
        for i in range(len(layout) - 1, -1, -1):
            if layout[i].isdigit():
                step += 8 * int(layout[i])
                continue
            strides[layout[i]] = step
            step *= extent[layout[i]]
        self.size = step
        self.strides = (strides["p"], strides["s"], strides["h"])
        self.k_bits = self.random_bits(self.size)
        self.v_bits = self.random_bits(self.size)
        self.geo = dict(heads=heads, kv_heads=kv, head_dim=dim, page_size=page, rotary_dim=kw.get("rotary_dim", dim) if kw.get("rotary_dim", dim) is not None else dim,
                        rope_base=kw.get("rope_base", 1e6), interleaved=kw.get("interleaved", False), norm_eps=kw.get("norm_eps", 1e-6))
        self.scale = kw.get("scale") or 1 / math.sqrt(dim)
        self.op = PagedAttention(heads, kv, dim, page_size=page, dtype=dtype, strides=self.strides, **kw)
        self.d_lens, self.d_table = hip.put(self.lens), hip.put(self.table)
        self.d_row0 = None if one_row else hip.put(self.row0)
        self.max_rows = max_rows
        self.batch = self.op.batch(self.d_lens, self.d_table, self.width, self.pages, len(seqs), rows=self.rows, row0=self.d_row0, max_rows=max_rows,
                                   table_stride=self.width + 2)
        self.kc = self.vc = None

    def random_bits(self, *shape, dtype=None):
        return O.to_bits(self.rng.standard_normal(shape, dtype=np.float32), dtype or self.dtype)

    def view(self, bits):
        """[pages][slots][heads][dim] view of a cache."""
        p, s, h = self.strides
        b = bits.itemsize
        return np.lib.stride_tricks.as_strided(bits, (self.pages, self.page, self.kv, self.dim), (p * b, s * b, h * b, b))

    def upload(self):
        self.kc, self.vc = self.hip.put(self.k_bits), self.hip.put(self.v_bits)

    def places(self):
        """Every (page, slot) that some sequence has."""
        return {O.slot(self.table[:, :self.width], self.pages, self.page, s, t) for s, n in enumerate(self.lens) for t in range(max(n, 0))} - {None}

    def attend(self, window=0, sinks=0, out_dtype=None, q_extra=0, out_extra=0, stream=None, q=None, check=True):
        out_dtype = out_dtype or self.dtype
        w = self.heads * self.dim
        if q is None:
            q = self.rng.standard_normal((self.rows, w + q_extra), dtype=np.float32) * (0.5 + 3 * self.rng.random((self.rows, 1), dtype=np.float32))
            q = O.to_bits(q, self.dtype)
        if self.kc is None:
            self.upload()
        guard = np.full((self.rows, w + out_extra), GUARD, np.uint16).astype(np.uint32 if out_dtype == "f32" else np.uint16)
        dq, do = self.hip.put(q), self.hip.put(guard)
        self.op.attend(self.batch, self.kc, self.vc, dq, do, out_dtype=out_dtype, window=window, sinks=sinks, q_stride=w + q_extra, out_stride=w + out_extra,
                       stream=stream)
        got = self.hip.get(do, guard)
        if check:
            self.check_attend(got, guard, q, window, sinks, out_dtype)
        return got

    def check_attend(self, got, guard, q, window, sinks, out_dtype):
        w = self.heads * self.dim
        qv = O.from_bits(q[:, :w], self.dtype).reshape(self.rows, self.heads, self.dim)
        with np.errstate(invalid="ignore", over="ignore"):
            ref, size, dots = O.attend(self.geo, self.lens, self.table[:, :self.width], self.row0, self.rows, self.pages, qv,
                                       O.from_bits(self.view(self.k_bits), self.dtype), O.from_bits(self.view(self.v_bits), self.dtype), window, sinks, self.scale)
        assert np.array_equal(got[:, w:], guard[:, w:]), "written between the rows"
        keep = [r for r in range(self.rows) if r not in ref]
        assert np.array_equal(got[keep], guard[keep]), "a row behind the last sequence was written"
        val = O.from_bits(got[:, :w], out_dtype) if out_dtype != "f32" else got[:, :w].view(np.float32).astype(np.float64)
        off2 = ref2 = 0.0
        h = O.HALF_STEP[out_dtype]
        weight = {"f16": 2.0 ** -22, "bf16": 2.0 ** -24}[self.dtype] if out_dtype == "f32" else O.HALF_STEP[self.dtype]
        n = int(self.lens.max(initial=1))
        for r in ref:
            y, g = ref[r], val[r].reshape(self.heads, self.dim)
            assert np.array_equal(np.isfinite(y), np.isfinite(g)), (r, np.argwhere(np.isfinite(y) != np.isfinite(g))[:4])
            f = np.isfinite(y)
            eta = dots[r] * (self.dim + 8) * U + 2.0 ** -21
            tol = h * np.abs(y) + (weight + 2 * eta + 2 * n * U) * size[r] + O.LEAST[out_dtype]
            bad = f & ~(np.abs(g - y) <= tol)
            assert not bad.any(), (r, np.argwhere(bad)[:4], g[bad][:4], y[bad][:4])
            off2 += float(((g - y)[f] ** 2).sum())
            ref2 += float((y[f] ** 2).sum())
        if ref2:
            assert math.sqrt(off2 / ref2) <= (1e-5 if out_dtype == "f32" else 1.5 * h)


# ---- append ------------------------------------------------------------------------------
APPEND = [
    # the engine's shape: one row, and prompts
    (dict(seqs=[(1, 1)], one_row=True), dict(x="f32", bias=True)),
    (dict(seqs=[(257, 1)], one_row=True), dict(x="f32", bias=True)),
    (dict(seqs=[(100, 37)]), dict(x="f16", bias=True)),
    # norms, both types, other layouts and pages
    (dict(seqs=[(5, 1), (64, 1), (65, 1), (1, 1), (900, 1)], heads=32, kv=8, dim=128, dtype="bf16", page=32, one_row=True), dict(norm=True)),
    (dict(seqs=[(40, 7), (3, 3), (33, 0), (700, 1), (130, 130)], heads=4, kv=4, dim=128, dtype="bf16", page=64, layout="phs", pad=5), dict(norm=True, x="f32")),
    (dict(seqs=[(40, 7), (3, 3), (33, 0), (700, 1)], heads=6, kv=1, dim=64, page=128, layout="p1h2s3", pad=2), dict(norm=True, bias=True)),
    (dict(seqs=[(40, 39), (41, 1)], heads=3, kv=3, dim=128, page=1024, layout="hps"), dict(x="f32")),
    # parts of the head, interleaved pairs, no rotation, other positions
    (dict(seqs=[(40, 39), (41, 1)], heads=4, kv=2, dim=64, rotary_dim=32), dict(bias=True)),
    (dict(seqs=[(40, 39), (41, 1)], heads=4, kv=2, dim=128, rotary_dim=80, interleaved=True, dtype="bf16"), dict(norm=True, x="f32")),
    (dict(seqs=[(40, 39), (41, 1)], heads=4, kv=2, dim=64, interleaved=True, rope_base=10000.0), dict(positions=True)),
    (dict(seqs=[(40, 39), (41, 1)], heads=4, kv=2, dim=64, rotary_dim=0), dict(norm=True)),
    (dict(seqs=[(40, 16), (41, 0), (17, 17)], heads=20, kv=1, dim=64, rotary_dim=16), dict(no_q=True, bias=True, norm=True)),
    # sequences without positions for all of their rows, empty ones, one that is longer than its table
    (dict(seqs=[(2, 5), (0, 2), (-7, 1), (0, 0), (18, 4)], pad=1), dict(norm=True)),
    # many sequences, so that a row's sequence is found over several steps
    (dict(seqs=[(i % 50 + 1, i % 4) for i in range(200)], heads=2, kv=1, dim=64), dict(x="f16")),
    (dict(seqs=[(i % 50 + 1, i % 4) for i in range(300)], heads=2, kv=2, dim=128, dtype="bf16", pad=3), dict(norm=True)),
    # prompts of which a workgroup takes several rows, the last one fewer
    (dict(seqs=[(1500, 1300), (2901, 2901)], heads=2, kv=1, pad=2), dict(norm=True, bias=True)),
    (dict(seqs=[(1031, 1031), (40, 1), (7, 9)], heads=3, kv=1, dim=128, dtype="bf16"), dict(x="f32")),
]


def _append(s, x="", bias=False, norm=False, positions=False, no_q=False, in_place=False, stream=None, extra=0):
    hip, x = s.hip, x or s.dtype
    heads, kv, dim, w = s.heads, s.kv, s.dim, s.heads * s.dim
    width = (heads + 2 * kv) * dim + extra
    xs = (s.random_bits(s.rows, width, dtype=x) if x != "f32" else s.rng.standard_normal((s.rows, width), dtype=np.float32))
    b = s.rng.standard_normal((heads + 2 * kv) * dim, dtype=np.float32) if bias else None
    qn, kn = [(1 + 0.2 * s.rng.standard_normal(dim, dtype=np.float32)).astype(np.float32) if norm else None for _ in range(2)]
    ps = s.rng.integers(-5, 1 << 30, s.rows).astype(np.int32) if positions else None
    guard = np.full((s.rows, w + 8), GUARD, np.uint16)
    if s.kc is None:
        s.upload()
    dx, do = hip.put(xs), hip.put(guard)
    dev = [None if a is None else hip.put(a) for a in (b, qn, kn, ps)]
    e = xs.itemsize
    out, stride = (dx, width) if in_place else (do, w + 8)
    s.op.append(s.batch, s.kc, s.vc, k=dx + e * w, v=dx + e * (w + kv * dim), q=None if no_q else dx, q_out=None if no_q else out, x_dtype=x, x_stride=width,
                q_out_stride=stride, bias=dev[0], q_norm=dev[1], k_norm=dev[2], positions=dev[3], stream=stream)
    got_q = hip.get(do, guard)
    if in_place:
        got_q = np.concatenate([hip.get(dx, xs)[:, :w], guard[:, w:]], 1)
        guard = np.concatenate([xs[:, :w], guard[:, w:]], 1)
    got_k, got_v = s.view(hip.get(s.kc, s.k_bits)), s.view(hip.get(s.vc, s.v_bits))
    xv = O.from_bits(xs[:, :width - extra], x).reshape(s.rows, heads + 2 * kv, dim)
    f = lambda a: None if a is None else a.astype(np.float64)   # noqa: E731
    queries, cached = O.append(s.geo, s.lens, s.table[:, :s.width], s.row0, s.rows, s.pages, xv[:, :heads], xv[:, heads:heads + kv], xv[:, heads + kv:], f(b),
                               f(qn), f(kn), ps)
    assert np.array_equal(got_q[:, w:], guard[:, w:]), "written between the rows"
    h, least = O.HALF_STEP[s.dtype], O.LEAST[s.dtype] / 2

    def close(bits, y, size, what):
        g = O.from_bits(np.ascontiguousarray(bits), s.dtype)
        bad = ~(np.abs(g - y) <= h * np.abs(y) + 32 * U * size + least)
        assert not bad.any(), (what, np.argwhere(bad)[:4], g[bad][:4], y[bad][:4])
    for r in range(s.rows):
        if no_q or r not in queries:
            assert np.array_equal(got_q[r], guard[r]), f"row {r} was written"
        else:
            close(got_q[r, :w].reshape(heads, dim), *queries[r], f"query {r}")
    rest_k, rest_v = s.view(s.k_bits.copy()), s.view(s.v_bits.copy())
    for (p, t), (key, size, val) in cached.items():
        close(got_k[p, t], key, size, f"key {p}, {t}")
        close(got_v[p, t], val, np.abs(val), f"value {p}, {t}")
        rest_k[p, t], rest_v[p, t] = got_k[p, t], got_v[p, t]
    # everything else in the buffers is as it was
    raw_k, raw_v = hip.get(s.kc, s.k_bits), hip.get(s.vc, s.v_bits)
    keep_k, keep_v = s.k_bits.copy(), s.v_bits.copy()
    s.view(keep_k)[...], s.view(keep_v)[...] = rest_k, rest_v
    assert np.array_equal(raw_k, keep_k) and np.array_equal(raw_v, keep_v), "the cache changed elsewhere"
    s.k_bits, s.v_bits = raw_k, raw_v
    return got_q, len(cached)


@pytest.mark.parametrize("setup,call", APPEND, ids=[str(i) for i in range(len(APPEND))])
def test_append_matches_oracle(hip, setup, call):
    print("append", setup, call, flush=True)
    _append(Setup(hip, **setup), **call)


def test_append_in_place_and_wide_rows(hip):
    s = Setup(hip, [(40, 39), (41, 1)], pad=3)
    _append(s, in_place=True, norm=True, bias=True)
    _append(s, extra=24, x="f32")


def test_append_far_positions(hip):
    """Positions up to 2^24 in a sequence: angles keep their fractions of a turn. Tables are wide, pages few."""
    n = 1 << 24
    s = Setup(hip, [(40, 33)], heads=2, kv=2, page=1024, spare=2)
    s.width = n // 1024
    s.table = np.zeros((1, s.width + 2), np.int32)
    s.lens[:] = n - 5
    hip.write(s.d_lens, s.lens)
    s.batch = s.op.batch(s.d_lens, hip.put(s.table), s.width, s.pages, 1, rows=s.rows, row0=s.d_row0, table_stride=s.width + 2)
    _append(s)


def test_append_bad_pages_and_short_tables(hip):
    """Rows whose page is out of range, or behind the table, are left out; their queries are turned all the same."""
    s = Setup(hip, [(70, 40), (30, 30), (16, 1)])
    s.table[0, 2], s.table[0, 3], s.table[1, 1] = -1, s.pages, 0x7FFFFFFF
    s.lens[2] = 16 * s.width + 1
    hip.write(s.d_table, s.table)
    hip.write(s.d_lens, s.lens)
    _, written = _append(s, norm=True)
    assert written == (2 + 6) + 16 + 0


# ---- attention ---------------------------------------------------------------------------
EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 500, 1000]
ATTEND = [
    # one new row each, lengths around the tiles' and pages' ends, and rows that see nothing
    (dict(seqs=[(n, 1) for n in EDGES], one_row=True, pad=2), dict()),
    (dict(seqs=[(n, 1) for n in EDGES], one_row=True, heads=32, kv=8, dim=128, dtype="bf16", page=32), dict()),
    (dict(seqs=[(n, 1) for n in EDGES], one_row=True, heads=3, kv=3, dim=64, dtype="bf16", page=1024, layout="phs"), dict(out_dtype="f32")),
    (dict(seqs=[(n, 1) for n in EDGES], heads=20, kv=1, dim=128, page=64, layout="hps"), dict(out_dtype="f32")),
    (dict(seqs=[(n, 1) for n in EDGES], heads=33, kv=1, dim=64, page=16, layout="p1s2h3", max_rows=1), dict(q_extra=8, out_extra=16)),
    # windows and sinks, one row each
    (dict(seqs=[(n, 1) for n in EDGES], one_row=True), dict(window=1)),
    (dict(seqs=[(n, 1) for n in EDGES], one_row=True), dict(window=16, sinks=1)),
    (dict(seqs=[(n, 1) for n in EDGES], one_row=True, heads=8, kv=2, dim=128, dtype="bf16"), dict(window=100, sinks=4)),
    (dict(seqs=[(n, 1) for n in EDGES], one_row=True, heads=8, kv=2, dim=128), dict(window=33, sinks=70, out_dtype="f32")),
    (dict(seqs=[(n, 1) for n in EDGES], one_row=True, page=256), dict(window=64, sinks=1 << 30)),
    (dict(seqs=[(n, 1) for n in EDGES], one_row=True), dict(window=(1 << 31) - 1, sinks=(1 << 31) - 1)),
    # a few new rows each (drafts), also more rows than positions
    (dict(seqs=[(500, 2), (100, 5), (16, 16), (3, 4), (0, 2), (77, 0), (260, 16), (-3, 1)], pad=3), dict()),
    (dict(seqs=[(500, 2), (100, 5), (16, 16), (3, 4), (260, 16)], heads=16, kv=2, dim=128, dtype="bf16", max_rows=16), dict(window=40, sinks=3)),
    (dict(seqs=[(500, 3), (100, 3), (16, 3)], heads=5, kv=5, max_rows=3), dict(out_dtype="f32")),
    # prompts, whole and behind cached positions, beside single rows
    (dict(seqs=[(1, 1), (130, 130), (257, 64), (300, 299), (90, 1)]), dict()),
    (dict(seqs=[(333, 333)]), dict(out_dtype="f32")),
    (dict(seqs=[(200, 129), (64, 64)], heads=8, kv=2, dim=128, dtype="bf16", page=64), dict()),
    (dict(seqs=[(200, 129), (64, 64), (31, 40)], heads=3, kv=3, dim=128, page=32, layout="phs", pad=4), dict(out_dtype="f32", q_extra=8, out_extra=4)),
    (dict(seqs=[(400, 400)], heads=4, kv=1), dict(window=50)),
    (dict(seqs=[(400, 300), (520, 200)], heads=7, kv=1, page=128, dtype="bf16"), dict(window=64, sinks=5)),
    (dict(seqs=[(400, 300), (520, 200)], heads=4, kv=2, dim=128), dict(window=17, sinks=100, out_dtype="f32")),
    (dict(seqs=[(700, 100)], heads=20, kv=1, dim=64), dict(window=1, sinks=1)),
    # long contexts, split over many workgroups
    (dict(seqs=[(9000, 1)], one_row=True), dict()),
    (dict(seqs=[(9001, 1), (40, 1)], one_row=True, heads=4, kv=1, dim=128, dtype="bf16"), dict(out_dtype="f32")),
    (dict(seqs=[(9001, 1), (7000, 1)], one_row=True, page=64), dict(window=5000, sinks=9)),
    (dict(seqs=[(5000, 40)], heads=4, kv=1), dict()),
    (dict(seqs=[(5000, 40), (3000, 90)], heads=4, kv=2, dim=128, dtype="bf16"), dict(out_dtype="f32", window=2500, sinks=300)),
    # enough tiles of 128 rows x heads for the prompt kernel: whole prompts, behind cached positions, windows, both head sizes and outputs
    (dict(seqs=[(333, 333)], heads=84, kv=84), dict()),
    (dict(seqs=[(200, 129), (64, 64), (31, 40), (1, 1)], heads=128, kv=64, dim=128, dtype="bf16", page=64, pad=2), dict(q_extra=8, out_extra=16)),
    (dict(seqs=[(400, 300)], heads=96, kv=32, layout="phs"), dict(window=50, sinks=5, out_dtype="f32")),
    (dict(seqs=[(700, 130)], heads=120, kv=120, dim=128, page=32), dict(window=1, sinks=1)),
    (dict(seqs=[(520, 200), (90, 90)], heads=72, kv=72, dtype="bf16", page=128, layout="p1h2s3"), dict(window=64, sinks=100)),
    (dict(seqs=[(300, 128), (129, 128)], heads=112, kv=112, dim=128, page=1024), dict(out_dtype="f32")),
    # both kernels, the prompt kernel's longest sequence in parts
    (dict(seqs=[(6000, 40)] + [(100 + i, 40) for i in range(7)] + [(900, 1), (64, 1), (0, 1), (5, 9), (70, 0)], heads=64, kv=32, pad=1), dict()),
    (dict(seqs=[(6000, 40)] + [(100 + i, 40) for i in range(7)] + [(900, 1), (64, 1), (0, 1), (5, 9), (70, 0)], heads=64, kv=32, dim=128, dtype="bf16", max_rows=40),
     dict(window=4500, sinks=70, out_dtype="f32")),
    # many sequences
    (dict(seqs=[(3 * i % 190, i % 3) for i in range(150)], heads=2, kv=1), dict(window=30, sinks=2)),
    (dict(seqs=[(7 * i % 300, 1) for i in range(130)], one_row=True, heads=4, kv=2, dim=128, scale=0.3), dict()),
    # more than a workgroup has threads, one of them in parts
    (dict(seqs=[(7 * i % 90, 1) if i != 290 else (6000, 1) for i in range(301)], one_row=True, heads=4, kv=2), dict()),
    (dict(seqs=[(25 + i % 9, 20) if i != 270 else (3000, 30) for i in range(280)] + [(9, 2), (70, 1)], heads=4, kv=2, pad=2), dict(sinks=2, window=2000)),
    # scores that leave only a few weights, with the greatest anywhere
    (dict(seqs=[(700, 1), (90, 5), (65, 1)], heads=4, kv=2, scale=4.0), dict()),
    (dict(seqs=[(300, 130), (129, 128)], heads=112, kv=112, dtype="bf16", scale=4.0), dict()),
]


@pytest.mark.parametrize("setup,call", ATTEND, ids=[str(i) for i in range(len(ATTEND))])
def test_attend_matches_oracle(hip, setup, call):
    print("attend", setup, call, flush=True)
    Setup(hip, **setup).attend(**call)


@pytest.mark.parametrize("dim,dtype", [(64, "f16"), (128, "bf16")])
@pytest.mark.parametrize("rows,heads,kv", [(1, 6, 2), (3, 6, 2), (40, 6, 2), (150, 6, 2), (150, 112, 112)], ids=["1", "3", "40", "150", "150-prompt-kernel"])
def test_what_is_not_seen_never_reaches_a_row(hip, dim, dtype, rows, heads, kv):
    """NaN and infinities in every slot that no sequence has, and in positions that only later rows, or rows before them (a window's), see."""
    s = Setup(hip, [(150, min(rows, 150)), (67, min(rows, 67)), (16, 1)], heads=heads, kv=kv, dim=dim, dtype=dtype)
    used = s.places()
    k, v = s.view(s.k_bits), s.view(s.v_bits)
    wild = O.to_bits(np.array([np.nan, np.inf, -np.inf], np.float32), dtype)
    for p in range(s.pages):
        for t in range(s.page):
            if (p, t) not in used:
                k[p, t], v[p, t] = s.rng.choice(wild, (2, s.kv, dim))
    s.attend()
    s.attend(window=20, sinks=3, out_dtype="f32")
    last = O.slot(s.table, s.pages, 16, 0, 149)
    early = O.slot(s.table, s.pages, 16, 0, 100)
    s.kc = None
    v[last[0], last[1], 0, 5:9] = O.to_bits(np.array([np.inf, -np.inf, np.nan, 1], np.float32), dtype)   # seen by the last row alone
    k[early[0], early[1], 1, 3] = wild[0]
    v[early[0], early[1], 1, 2] = wild[1]
    s.attend()
    s.attend(window=20, sinks=3, out_dtype="f32")


@pytest.mark.parametrize("heads,kv", [(4, 2), (228, 228)], ids=["step", "both"])
def test_attend_bad_pages(hip, heads, kv):
    """Positions on pages out of range are not seen."""
    s = Setup(hip, [(300, 1), (300, 60), (40, 2)], heads=heads, kv=kv)
    s.table[0, 3], s.table[0, 18], s.table[1, 0], s.table[1, 17], s.table[2, :3] = -1, s.pages, 0x7FFFFFFF, -0x80000000, -5
    hip.write(s.d_table, s.table)
    s.attend()
    s.attend(window=70, sinks=20, out_dtype="f32")


@pytest.mark.parametrize("heads,kv", [(4, 2), (232, 116)], ids=["step", "both"])
def test_attend_lengths_past_the_table(hip, heads, kv):
    """Positions behind the table's last page are not seen; the rows stand where the length says."""
    s = Setup(hip, [(48, 1), (48, 30), (40, 20)], heads=heads, kv=kv)
    s.lens[:] = [60, 70, 200]
    hip.write(s.d_lens, s.lens)
    s.attend()
    s.attend(window=25, sinks=2)


def test_pages_shared_by_sequences(hip):
    s = Setup(hip, [(100, 1), (90, 20), (64, 1)], heads=4, kv=2)
    s.table[1, :3] = s.table[0, :3]
    s.table[2, :4] = s.table[0, 0]
    hip.write(s.d_table, s.table)
    s.attend()


def test_offsets_past_32_bits(hip):
    """Pages 2^27 elements apart: the last ones begin past 2^31 elements (2^32 bytes)."""
    from instantllm_amd.paged import PagedAttention
    heads, kv, dim, page, step, pages = 4, 2, 64, 16, 1 << 27, 20
    rng = np.random.default_rng(5)
    small = Setup(hip, [(60, 1), (61, 33)], heads=heads, kv=kv, spare=pages - 8, seed=3, shuffle=False)
    assert small.pages == pages
    small.table[0, :4], small.table[1, :4] = [19, 0, 18, 17], [16, 2, 3, 15]
    hip.write(small.d_table, small.table)
    q = O.to_bits(rng.standard_normal((34, heads * dim), dtype=np.float32), "f16")
    expect = small.attend(q=q)
    big = [hip.alloc(2 * step * pages) for _ in range(2)]
    for addr, bits in zip(big, (small.k_bits, small.v_bits)):
        for p in range(pages):
            hip.write(addr + 2 * step * p, small.view(bits)[p])
    op = PagedAttention(heads, kv, dim, page_size=page, strides=(step, kv * dim, dim))
    out = hip.put(np.zeros_like(expect))
    b = op.batch(small.d_lens, small.d_table, small.width, pages, 2, rows=34, row0=small.d_row0, table_stride=small.width + 2)
    op.attend(b, *big, hip.put(q), out)
    assert np.array_equal(hip.get(out, expect), expect)
    x = rng.standard_normal((34, (heads + 2 * kv) * dim), dtype=np.float32)
    dx, w = hip.put(x), heads * dim
    kw = dict(k=dx + 4 * w, v=dx + 4 * (w + kv * dim), x_dtype="f32", x_stride=(heads + 2 * kv) * dim)
    op.append(b, *big, **kw)
    small.op.append(small.batch, small.kc, small.vc, **kw)
    for addr, ref, bits in zip(big, (small.kc, small.vc), (small.k_bits, small.v_bits)):
        want = small.view(hip.get(ref, bits))
        for p in (2, 15, 16, 17, 18, 19):
            assert np.array_equal(hip.get(addr + 2 * step * p, want[p]), want[p])


def test_attend_is_deterministic_and_independent_of_earlier_calls(hip):
    """The same call's bits, also after calls of other sizes on the same handle."""
    s = Setup(hip, [(9000, 1), (300, 40), (1, 1)], heads=112, kv=112)
    q = s.random_bits(42, s.heads * s.dim)
    first = s.attend(q=q, check=False)
    for _ in range(3):
        s.attend(window=4000, sinks=3, check=False)
        assert np.array_equal(s.attend(q=q, check=False), first)


# ---- together ----------------------------------------------------------------------------
def _layer(s, hip, x, stream):
    """Append and attention of one layer on a stream; returns the addresses of the queries and outputs."""
    heads, kv, dim, w = s.heads, s.kv, s.dim, s.heads * s.dim
    q, out = hip.alloc(2 * s.rows * w), hip.alloc(4 * s.rows * w)

    def enqueue():
        s.op.append(s.batch, s.kc, s.vc, k=x + 4 * w, v=x + 4 * (w + kv * dim), q=x, q_out=q, x_dtype="f32", x_stride=(heads + 2 * kv) * dim, stream=stream)
        s.op.attend(s.batch, s.kc, s.vc, q, out, out_dtype="f32", stream=stream)
    return enqueue, q, out


def test_graphs_follow_lengths_and_tables(hip):
    """A captured layer replayed over growing sequences equals the eager calls; two graphs of one handle, and eager calls between them."""
    s = Setup(hip, [(4000, 1), (130, 1), (15, 1)], one_row=True, spare=0)
    twin = Setup(hip, [(4000, 1), (130, 1), (15, 1)], one_row=True, spare=0)
    for z in (s, twin):
        z.lens -= 9
        z.upload()
    st = [hip.stream(), hip.stream()]
    xs = [s.rng.standard_normal((3, 18 * 64), dtype=np.float32) for _ in range(9)]
    x, xt = hip.put(xs[0]), hip.put(xs[0])
    layers = [_layer(s, hip, x, st[i]) for i in range(2)]
    eager, tq, tout = _layer(twin, hip, xt, None)
    graphs = [hip.capture(st[i], layers[i][0]) for i in range(2)]
    for step, data in enumerate(xs):
        for z, dst in ((s, x), (twin, xt)):
            z.lens += 1
            hip.write(z.d_lens, z.lens)
            hip.write(dst, data)
        hip.sync()
        for i in range(2):   # the second graph appends the same rows again
            hip.launch(graphs[i], st[i])
            hip.sync()
        eager()
        want = hip.get(tout, np.zeros((3, 14 * 64), np.float32))
        for _, q, out in layers:
            assert np.array_equal(hip.get(out, want), want), step
            assert np.array_equal(hip.get(q, np.zeros((3, 14 * 64), np.uint16)), hip.get(tq, np.zeros((3, 14 * 64), np.uint16)))
        s.attend(check=False)   # an eager call of another size between the replays
    assert np.array_equal(hip.get(s.kc, s.k_bits), hip.get(twin.kc, s.k_bits))


def test_graphs_at_once(hip):
    """Two graphs of a batch that both kernels and split keys take part in, and an eager call, at a time and again."""
    s = Setup(hip, [(6000, 40)] + [(100 + i, 40) for i in range(7)] + [(900, 1), (64, 1), (0, 1), (5, 9), (70, 0)], heads=64, kv=32)
    s.upload()
    w = s.heads * s.dim
    qs = [s.random_bits(s.rows, w) for _ in range(3)]
    want = [s.attend(q=q) for q in qs]
    st = [hip.stream(), hip.stream(), None]
    dq, do = [hip.put(q) for q in qs], [hip.alloc(2 * s.rows * w) for _ in st]
    calls = [lambda i=i: s.op.attend(s.batch, s.kc, s.vc, dq[i], do[i], stream=st[i]) for i in range(3)]
    graphs = [hip.capture(st[i], calls[i]) for i in range(2)]
    for turn in range(5):
        for i in range(3):
            hip.write(do[i], np.zeros_like(want[i]))
        hip.sync()
        for _ in range(2):
            for i in range(2):
                hip.launch(graphs[i], st[i])
            calls[2]()
        for i in range(3):
            assert np.array_equal(hip.get(do[i], want[i]), want[i]), (turn, i)


def test_rows_before_the_first_sequence(hip):
    """Rows in front of row0[0] are no sequence's: neither call writes them."""
    s = Setup(hip, [(70, 3), (5, 0), (300, 40)], pad=1)
    s.row0 += 2
    s.rows += 2
    hip.write(s.d_row0, s.row0)
    s.batch = s.op.batch(s.d_lens, s.d_table, s.width, s.pages, 3, rows=s.rows, row0=s.d_row0, table_stride=s.width + 2)
    _append(s, bias=True)
    s.attend()


def test_streams_at_once(hip):
    """Calls of one handle on several streams at a time keep apart."""
    s = Setup(hip, [(9000, 1)], one_row=True)
    s.upload()
    st = [hip.stream() for _ in range(3)]
    w = s.heads * s.dim
    qs = [s.random_bits(1, w) for _ in st]
    want = [s.attend(q=q) for q in qs]
    dq, do = [hip.put(q) for q in qs], [hip.alloc(2 * w) for _ in st]
    for _ in range(10):
        for i in range(3):
            s.op.attend(s.batch, s.kc, s.vc, dq[i], do[i], stream=st[i])
    for i in range(3):
        assert np.array_equal(hip.get(do[i], want[i]), want[i])


def test_an_attention_block_with_the_stand_alone_product(hip):
    """QKV product, append, attention and output product of the engine's shape over a growing sequence, against float64."""
    from instantllm_amd import synth
    from instantllm_amd.engine import Gemv
    from oracle import illread
    s = Setup(hip, [(30, 1)], one_row=True)
    s.lens[:] = 0
    s.upload()
    mats = []
    for seed, rows, k in ((1, 1152, 896), (2, 896, 896)):
        codes, sb = synth.microbench_q4(seed, rows, k)
        mats.append((Gemv(codes, np.ascontiguousarray(sb).view(np.uint32).reshape(rows, k // 64)), illread.dequant_q4(codes, sb).astype(np.float64)))
    bias = s.rng.standard_normal(1152, dtype=np.float32)
    d_bias, d_x, d_qkv, d_q, d_att, d_y = hip.put(bias), hip.alloc(4 * 896), hip.alloc(4 * 1152), hip.alloc(2 * 896), hip.alloc(4 * 896), hip.alloc(4 * 896)
    stream = hip.stream()
    keys, vals = np.zeros((0, 2, 64)), np.zeros((0, 2, 64))
    for t in range(30):
        x = synth.microbench_x(t, 896)[0][0].astype(np.float32)
        s.lens[:] = t + 1
        hip.write(s.d_lens, s.lens)
        hip.write(d_x, x)
        hip.sync()
        mats[0][0].run_noalloc(d_x, None, d_qkv, None, stream=stream)
        s.op.append(s.batch, s.kc, s.vc, k=d_qkv + 4 * 896, v=d_qkv + 4 * 1024, q=d_qkv, q_out=d_q, x_dtype="f32", bias=d_bias, stream=stream)
        s.op.attend(s.batch, s.kc, s.vc, d_q, d_att, out_dtype="f32", stream=stream)
        mats[1][0].run_noalloc(d_att, None, d_y, None, stream=stream)
        y = hip.get(d_y, np.zeros(896, np.float32)).astype(np.float64)
        qkv = (mats[0][1] @ x + bias).reshape(18, 64)
        q, _ = O.turn(qkv[:14], t, 64, 1e6, False)
        k, _ = O.turn(qkv[14:16], t, 64, 1e6, False)
        keys, vals = np.concatenate([keys, k[None]]), np.concatenate([vals, qkv[None, 16:]])
        att = np.zeros((14, 64))
        for h in range(14):
            sc = keys[:, h // 7] @ q[h] / 8
            p = np.exp(sc - sc.max())
            att[h] = p @ vals[:, h // 7] / p.sum()
        ref = mats[1][1] @ att.reshape(-1)
        # the decode step's tolerance: products in 16-bit fixed point, queries, keys and values rounded to f16
        assert np.linalg.norm(y - ref) <= 1e-2 * np.linalg.norm(ref), t


@pytest.mark.parametrize("max_rows", [1, 3, 1 << 40])
def test_a_wrong_hint_of_the_most_rows(hip, max_rows):
    """max_rows only chooses kernels: too small or too large, every row is evaluated."""
    s = Setup(hip, [(200, 129), (64, 64), (31, 40), (1, 1)], heads=64, kv=64, max_rows=max_rows)
    s.attend()


def test_workspaces_run_out_and_are_released(hip):
    from instantllm_amd.engine import ILL_E_ARG, IllError
    s = Setup(hip, [(9000, 1)], one_row=True, streams=2)
    s.upload()
    st = [hip.stream() for _ in range(2)]
    dq, do = hip.put(s.random_bits(1, 896)), hip.alloc(2 * 896)
    for stream in (st[0], None, st[0]):
        s.op.attend(s.batch, s.kc, s.vc, dq, do, stream=stream)
    with pytest.raises(IllError, match="ill_paged_release") as e:
        s.op.attend(s.batch, s.kc, s.vc, dq, do, stream=st[1])
    assert e.value.code == ILL_E_ARG
    hip.sync()
    s.op.release()
    s.op.attend(s.batch, s.kc, s.vc, dq, do, stream=st[1])
    s.attend(stream=st[0])


def test_the_per_thread_stream_is_refused(hip):
    from instantllm_amd.engine import IllError
    s = Setup(hip, [(3, 1)], one_row=True)
    s.upload()
    with pytest.raises(IllError, match="per-thread"):
        s.op.attend(s.batch, s.kc, s.vc, s.kc, s.vc, stream=2)


def test_nothing_to_do(hip):
    s = Setup(hip, [(3, 1)], one_row=True)
    s.upload()
    out = hip.put(np.full(896, GUARD, np.uint16))
    for b in (s.op.batch(s.d_lens, s.d_table, 1, s.pages, 0, rows=3), s.op.batch(s.d_lens, s.d_table, 1, s.pages, 1, rows=0, row0=s.d_row0 or s.d_lens)):
        s.op.attend(b, s.kc, s.vc, s.kc, out)
        s.op.append(b, s.kc, s.vc, k=s.vc, v=s.vc)
    assert (hip.get(out, np.zeros(896, np.uint16)) == GUARD).all()
    assert np.array_equal(hip.get(s.kc, s.k_bits), s.k_bits)
