"""GPU tests of paged caches of microscaled 8-bit keys and values, and of rows read out of either kind of cache, against the float64
restatements (oracle/paged.py, oracle/mx.py).

Attention multiplies the cache's values as values of the handle's type (exact in bf16; f16 rounds what lies below 2^-14), so
its tolerances are those of a 16-bit cache that holds them (test_gpu_paged.py).
append: a key is computed in float32, off by at most 32 u z (test_gpu_paged.py), and then rounded once to its block's codes: what
the cache holds lies between what the ends of that interval are held as, under a power that one of the interval's ends gives its block's
largest size. Values without a bias are not computed with: they are held as the restatement's, bit for bit.
"""
from __future__ import annotations

import numpy as np
import pytest

from hip_buffers import Hip
from oracle import mx as M
from oracle import paged as O
from test_gpu_paged import APPEND, ATTEND, GUARD, U, Setup

pytestmark = pytest.mark.gpu


@pytest.fixture()
def hip():
    h = Hip()
    yield h
    h.close()


class MxSetup(Setup):
    """A Setup whose caches are microscaled: bytes [pages][page_stride]. gap: bytes between pages."""

    def __init__(self, hip, seqs, layout=None, gap=0, streams=8, **kw):
        from instantllm_amd.paged import PagedAttention
        super().__init__(hip, seqs, streams=streams, **kw)
        self.op.close()
        call = {k: v for k, v in kw.items() if k in ("rotary_dim", "rope_base", "interleaved", "norm_eps", "scale")}
        n = self.page * self.kv * self.dim
        self.codes = n
        self.page_stride = n + n // 32 + gap
        self.op = PagedAttention(self.heads, self.kv, self.dim, page_size=self.page, dtype=self.dtype, cache="mxf8", streams=streams,
                                 page_stride=self.page_stride if gap else None, **call)
        assert self.op.page_bytes == n + n // 32
        self.k_bits, self.v_bits = self.random_cache(), self.random_cache()

    def random_cache(self):
        """Codes of sizes from 2^-3 to 448, either sign; powers around 2^-8; anything between the pages."""
        c = self.rng.integers(0, 256, (self.pages, self.page_stride), dtype=np.uint8)
        n = self.codes
        c[:, :n] = self.rng.integers(0x20, 0x7F, (self.pages, n)) | (c[:, :n] & 128)
        c[:, n:n + n // 32] = self.rng.integers(117, 121, (self.pages, n // 32))
        return c

    def parts(self, cache):
        """(codes [pages][kv][page][dim], powers [pages][kv][page][dim / 32]), views."""
        n = self.codes
        return (cache[:, :n].reshape(self.pages, self.kv, self.page, self.dim), cache[:, n:n + n // 32].reshape(self.pages, self.kv, self.page, self.dim // 32))

    def values(self, cache):
        """[pages][page][kv][dim] in float64."""
        return M.values(*(np.ascontiguousarray(p) for p in self.parts(cache)), "mxf8").transpose(0, 2, 1, 3)

    def view(self, cache):
        with np.errstate(over="ignore"):
            return O.to_bits(self.values(cache).astype(np.float32), self.dtype)


# ---- append and read ---------------------------------------------------------------------
def _append(s, x="", bias=False, norm=False, positions=False, no_q=False, stream=None, values=None):
    hip, x = s.hip, x or s.dtype
    heads, kv, dim, w = s.heads, s.kv, s.dim, s.heads * s.dim
    width = (heads + 2 * kv) * dim
    xs = s.rng.standard_normal((s.rows, width), dtype=np.float32) * np.exp2(s.rng.integers(-6, 6, (s.rows, 1))).astype(np.float32)
    if values is not None:
        values(xs)
    xs = O.to_bits(xs, x)
    b = s.rng.standard_normal(width, dtype=np.float32) if bias else None
    qn, kn = [(1 + 0.2 * s.rng.standard_normal(dim, dtype=np.float32)).astype(np.float32) if norm else None for _ in range(2)]
    ps = s.rng.integers(-5, 1 << 30, s.rows).astype(np.int32) if positions else None
    guard = np.full((s.rows, w + 8), GUARD, np.uint16)
    if s.kc is None:
        s.upload()
    dx, do = hip.put(xs), hip.put(guard)
    dev = [None if a is None else hip.put(a) for a in (b, qn, kn, ps)]
    e = xs.itemsize
    s.op.append(s.batch, s.kc, s.vc, k=dx + e * w, v=dx + e * (w + kv * dim), q=None if no_q else dx, q_out=None if no_q else do, x_dtype=x, x_stride=width,
                q_out_stride=w + 8, bias=dev[0], q_norm=dev[1], k_norm=dev[2], positions=dev[3], stream=stream)
    got_q, raw_k, raw_v = hip.get(do, guard), hip.get(s.kc, s.k_bits), hip.get(s.vc, s.v_bits)
    xv = O.from_bits(xs, x).reshape(s.rows, heads + 2 * kv, dim)
    f = lambda a: None if a is None else a.astype(np.float64)   # noqa: E731
    with np.errstate(invalid="ignore"):
        queries, cached = O.append(s.geo, s.lens, s.table[:, :s.width], s.row0, s.rows, s.pages, xv[:, :heads], xv[:, heads:heads + kv], xv[:, heads + kv:], f(b),
                                   f(qn), f(kn), ps)
    h, least = O.HALF_STEP[s.dtype], O.LEAST[s.dtype] / 2
    assert np.array_equal(got_q[:, w:], guard[:, w:])
    for r in range(s.rows):
        if no_q or r not in queries:
            assert np.array_equal(got_q[r], guard[r]), f"row {r} was written"
        else:
            y, size = queries[r]
            g = O.from_bits(np.ascontiguousarray(got_q[r, :w]), s.dtype).reshape(heads, dim)
            with np.errstate(invalid="ignore"):
                assert (np.isnan(y) | (np.abs(g - y) <= h * np.abs(y) + 32 * U * size + least)).all(), f"query {r}"
    # the cache: what has to be there, and everything else as it was
    want_k, want_v = s.k_bits.copy(), s.v_bits.copy()
    (gk, gkp), (gv, gvp), (wk, wkp), (wv, wvp) = (s.parts(c) for c in (raw_k, raw_v, want_k, want_v))
    for (p, t), (key, size, val) in cached.items():
        if b is None:
            c, e = M.quantize(val, "mxf8")
            assert np.array_equal(gv[p, :, t], c) and np.array_equal(gvp[p, :, t], e), f"value {p}, {t}"
        else:
            _between(gv[p, :, t], gvp[p, :, t], val, 2 * U * np.abs(val), f"value {p}, {t}")
        _between(gk[p, :, t], gkp[p, :, t], key, 32 * U * size, f"key {p}, {t}")
        wk[p, :, t], wkp[p, :, t], wv[p, :, t], wvp[p, :, t] = gk[p, :, t], gkp[p, :, t], gv[p, :, t], gvp[p, :, t]
    assert np.array_equal(raw_k, want_k) and np.array_equal(raw_v, want_v), "the cache changed elsewhere"
    s.k_bits, s.v_bits = raw_k, raw_v
    return len(cached)


def _between(codes, powers, y, off, what):
    codes, powers = np.ascontiguousarray(codes), np.ascontiguousarray(powers)
    blocks = np.abs(y).reshape(*powers.shape, 32)
    bad = ~np.isfinite(blocks).all(-1)
    assert np.array_equal(powers == 255, bad), what
    if bad.any():
        assert (codes.reshape(*powers.shape, 32)[bad] == 0).all()
        keep = ~bad
        codes, y, off = (a.reshape(*powers.shape, 32)[keep].reshape(-1, 32) for a in (codes, y, off))
        powers, blocks = powers[keep].reshape(-1, 1), blocks[keep].reshape(-1, 1, 32)
    d = off.reshape(*powers.shape, 32)
    ends = [M.quantize((blocks + sign * d).clip(0).max(-1, keepdims=True).repeat(32, -1).reshape(*powers.shape[:-1], -1), "mxf8")[1] for sign in (-1, 1)]
    assert ((powers >= ends[0]) & (powers <= ends[1])).all(), (what, powers, ends)
    g = M.values(codes, powers, "mxf8")
    assert ((g >= M.held_as(y - off, powers, "mxf8")) & (g <= M.held_as(y + off, powers, "mxf8"))).all(), what


MX_APPEND = [({k: v for k, v in s.items() if k != "layout"}, c) for s, c in APPEND]


@pytest.mark.parametrize("setup,call", MX_APPEND, ids=[str(i) for i in range(len(MX_APPEND))])
def test_append_matches_oracle(hip, setup, call):
    print("append", setup, call, flush=True)
    _append(MxSetup(hip, gap=48 * (len(setup["seqs"]) % 2), **setup), **call)


@pytest.mark.parametrize("dim,rotary", [(64, 0), (64, 16), (64, 48), (128, 16), (128, 48), (128, 112)])
def test_append_blocks_across_the_rotation(hip, dim, rotary):
    """Rotated and other dims in one block, pairs in two."""
    for interleaved in (False, True):
        _append(MxSetup(hip, [(40, 20), (33, 3)], heads=4, kv=2, dim=dim, rotary_dim=rotary, interleaved=interleaved, dtype="bf16"), norm=True)


def test_append_of_infinities_and_zeros(hip):
    """An infinity or NaN makes its block of 32 one of NaN; zeros, the least and the largest numbers."""
    def values(xs):
        w = 4 * 64
        xs[3, w + 5], xs[4, w + 2 * 64 + 40], xs[5, w + 3 * 64 + 1] = np.nan, np.inf, -np.inf
        xs[6] = 0
        xs[7, w + 2 * 64:] = 2.0 ** -149
        xs[8, w + 2 * 64 + 7] = 3.4e38
        xs[9, w + 2 * 64:] = 2.0 ** -126
    for x in ("f32", ""):
        _append(MxSetup(hip, [(40, 20), (33, 3)], heads=4, kv=2, dim=64, dtype="bf16", rotary_dim=0), x=x, values=values)


def test_append_bad_pages_and_short_tables(hip):
    s = MxSetup(hip, [(70, 40), (30, 30), (16, 1)])
    s.table[0, 2], s.table[0, 3], s.table[1, 1] = -1, s.pages, 0x7FFFFFFF
    s.lens[2] = 16 * s.width + 1
    hip.write(s.d_table, s.table)
    hip.write(s.d_lens, s.lens)
    assert _append(s, norm=True) == (2 + 6) + 16 + 0


def _read(s, dtype, extra=0, stream=None):
    kw = s.kv * s.dim
    guard = np.full((s.rows, kw + extra), GUARD, np.uint32 if dtype == "f32" else np.uint16)
    if s.kc is None:
        s.upload()
    out = [s.hip.put(guard) for _ in range(2)]
    s.op.read(s.batch, s.kc, s.vc, *out, dtype=dtype, k_stride=kw + extra, v_stride=kw + extra, stream=stream)
    for d, bits in zip(out, (s.k_bits, s.v_bits)):
        got, want = s.hip.get(d, guard), guard.copy()
        if isinstance(s, MxSetup):
            v = s.values(bits).astype(np.float32)
        else:
            v = O.from_bits(np.ascontiguousarray(s.view(bits)), s.dtype).astype(np.float32)
        for r, q, t in O.rows_of(s.lens, s.row0, s.rows):
            at = O.slot(s.table[:, :s.width], s.pages, s.page, q, t)
            y = np.zeros(kw, np.float32) if at is None else v[at].reshape(-1)
            with np.errstate(over="ignore"):
                want[r, :kw] = O.to_bits(y, dtype).view(want.dtype)
        a, b = (O.from_bits(np.ascontiguousarray(z), dtype) if dtype != "f32" else np.ascontiguousarray(z).view(np.float32) for z in (got, want))
        assert np.array_equal(a, b, equal_nan=True) and np.array_equal(got[:, kw:], guard[:, kw:])


READ = [(dict(seqs=[(1, 1)], one_row=True), 0), (dict(seqs=[(n, n) for n in (0, 1, 15, 16, 17, 300, 33)], pad=2), 8),
        (dict(seqs=[(500, 500), (40, 3), (70, 0), (2, 5), (-3, 1)], heads=32, kv=8, dim=128, dtype="bf16", page=32), 0),
        (dict(seqs=[(700, 650)], heads=3, kv=3, dim=128, page=1024, dtype="bf16"), 16),
        (dict(seqs=[(i % 50 + 1, i % 4) for i in range(300)], heads=2, kv=2, dim=64, dtype="bf16", pad=3), 0),
        (dict(seqs=[(1500, 1300), (2901, 2901)], heads=4, kv=4, pad=2), 0)]


@pytest.mark.parametrize("mx", [True, False], ids=["mxf8", "16-bit"])
@pytest.mark.parametrize("setup,extra", READ, ids=[str(i) for i in range(len(READ))])
def test_read_matches_cache(hip, setup, extra, mx):
    print("read", setup, extra, mx, flush=True)
    s = (MxSetup if mx else Setup)(hip, **setup)
    if mx:   # every code and power
        codes, powers = s.parts(s.k_bits)
        codes[...] = s.rng.integers(0, 256, codes.shape, dtype=np.uint8)
        powers[...] = s.rng.integers(0, 256, powers.shape, dtype=np.uint8)
    elif s.pages * s.page > 1000:
        s = Setup(hip, layout="phs", **setup)
    for dtype in (s.dtype, "f32"):
        _read(s, dtype, extra)


def test_read_bad_pages(hip):
    for kind in (MxSetup, Setup):
        s = kind(hip, [(70, 70), (30, 30), (16, 2)])
        s.table[0, 2], s.table[0, 3], s.table[1, 1] = -1, s.pages, 0x7FFFFFFF
        s.lens[2] = 16 * s.width + 1
        hip.write(s.d_table, s.table)
        hip.write(s.d_lens, s.lens)
        _read(s, s.dtype)


# ---- attention ---------------------------------------------------------------------------
MX_ATTEND = [({k: v for k, v in s.items() if k != "layout"}, c) for s, c in ATTEND]


@pytest.mark.parametrize("setup,call", MX_ATTEND, ids=[str(i) for i in range(len(MX_ATTEND))])
def test_attend_matches_oracle(hip, setup, call):
    print("attend", setup, call, flush=True)
    MxSetup(hip, gap=16 * (len(setup["seqs"]) % 3), **setup).attend(**call)


@pytest.mark.parametrize("dim,dtype", [(64, "f16"), (128, "bf16")])
@pytest.mark.parametrize("rows,heads,kv", [(1, 6, 2), (3, 6, 2), (40, 6, 2), (150, 6, 2), (150, 112, 112)], ids=["1", "3", "40", "150", "150-prompt-kernel"])
def test_what_is_not_seen_never_reaches_a_row(hip, dim, dtype, rows, heads, kv):
    """NaN blocks, NaN codes and powers that leave the type's range in every slot that no sequence has, and in positions that only
    later rows, or rows before them (a window's), see."""
    s = MxSetup(hip, [(150, min(rows, 150)), (67, min(rows, 67)), (16, 1)], heads=heads, kv=kv, dim=dim, dtype=dtype)
    used = s.places()
    (k, kp), (v, vp) = s.parts(s.k_bits), s.parts(s.v_bits)
    for p in range(s.pages):
        for t in range(s.page):
            if (p, t) not in used:
                kp[p, :, t], vp[p, :, t] = s.rng.choice([255, 254, 120], (2, kv, dim // 32))
                k[p, :, t], v[p, :, t] = s.rng.choice([0x7F, 0xFF, 0x7E, 0xFE], (2, kv, dim))
    s.attend()
    s.attend(window=20, sinks=3, out_dtype="f32")
    last = O.slot(s.table, s.pages, 16, 0, 149)
    early = O.slot(s.table, s.pages, 16, 0, 100)
    s.kc = None
    v[last[0], 0, last[1], 5] = 0x7F   # seen by the last row alone
    vp[last[0], 0, last[1], 1] = 255
    kp[early[0], 1, early[1], 0] = 255
    if dtype == "f16":   # infinite there
        vp[last[0], 1, last[1], 1] = 150
        v[early[0], 1, early[1], 2] = 0x7E
        vp[early[0], 1, early[1], 0] = 140
    s.attend()
    s.attend(window=20, sinks=3, out_dtype="f32")


@pytest.mark.parametrize("heads,kv", [(4, 2), (228, 228)], ids=["step", "both"])
def test_attend_bad_pages(hip, heads, kv):
    s = MxSetup(hip, [(300, 1), (300, 60), (40, 2)], heads=heads, kv=kv)
    s.table[0, 3], s.table[0, 18], s.table[1, 0], s.table[1, 17], s.table[2, :3] = -1, s.pages, 0x7FFFFFFF, -0x80000000, -5
    hip.write(s.d_table, s.table)
    s.attend()
    s.attend(window=70, sinks=20, out_dtype="f32")


@pytest.mark.parametrize("heads,kv", [(4, 2), (232, 116)], ids=["step", "both"])
def test_attend_lengths_past_the_table(hip, heads, kv):
    s = MxSetup(hip, [(48, 1), (48, 30), (40, 20)], heads=heads, kv=kv)
    s.lens[:] = [60, 70, 200]
    hip.write(s.d_lens, s.lens)
    s.attend()
    s.attend(window=25, sinks=2)


def test_pages_shared_by_sequences(hip):
    s = MxSetup(hip, [(100, 1), (90, 20), (64, 1)], heads=4, kv=2)
    s.table[1, :3] = s.table[0, :3]
    s.table[2, :4] = s.table[0, 0]
    hip.write(s.d_table, s.table)
    s.attend()


@pytest.mark.parametrize("heads,kv,dim,dtype", [(14, 2, 64, "f16"), (112, 112, 128, "bf16")])
def test_tiny_and_wide_powers(hip, heads, kv, dim, dtype):
    """Blocks of subnormal codes and of powers far apart, also where f16 has only subnormals for them."""
    s = MxSetup(hip, [(200, 130), (90, 1)], heads=heads, kv=kv, dim=dim, dtype=dtype)
    for cache in (s.k_bits, s.v_bits):
        codes, powers = s.parts(cache)
        codes[:, :, ::3] &= 0x87
        powers[...] = s.rng.choice([1, 90, 105, 112, 119, 121], powers.shape)
    s.attend()
    s.attend(out_dtype="f32")


def test_offsets_past_32_bits(hip):
    """Pages 2^28 bytes apart: the last ones begin past 2^32 bytes."""
    from instantllm_amd.paged import PagedAttention
    heads, kv, dim, page, step, pages = 4, 2, 64, 16, 1 << 28, 20
    small = MxSetup(hip, [(60, 1), (61, 33)], heads=heads, kv=kv, spare=pages - 8, seed=3, shuffle=False)
    assert small.pages == pages
    small.table[0, :4], small.table[1, :4] = [19, 0, 18, 17], [16, 2, 3, 15]
    hip.write(small.d_table, small.table)
    rng = np.random.default_rng(5)
    q = O.to_bits(rng.standard_normal((34, heads * dim), dtype=np.float32), "f16")
    expect = small.attend(q=q)
    big = [hip.alloc(step * pages) for _ in range(2)]
    for addr, bits in zip(big, (small.k_bits, small.v_bits)):
        for p in range(pages):
            hip.write(addr + step * p, bits[p])
    op = PagedAttention(heads, kv, dim, page_size=page, cache="mxf8", page_stride=step)
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
        want = hip.get(ref, bits)
        for p in (2, 15, 16, 17, 18, 19):
            assert np.array_equal(hip.get(addr + step * p, want[p]), want[p])
    like = np.empty((34, kv * dim), np.float32)
    outs = [hip.alloc(like.nbytes) for _ in range(4)]
    op.read(b, *big, *outs[:2], dtype="f32")
    small.op.read(small.batch, small.kc, small.vc, *outs[2:], dtype="f32")
    for i in range(2):
        assert np.array_equal(hip.get(outs[i], like), hip.get(outs[2 + i], like))


def test_attend_is_deterministic_and_independent_of_earlier_calls(hip):
    s = MxSetup(hip, [(9000, 1), (300, 40), (1, 1)], heads=112, kv=112)
    q = s.random_bits(42, s.heads * s.dim)
    first = s.attend(q=q, check=False)
    for _ in range(3):
        s.attend(window=4000, sinks=3, check=False)
        assert np.array_equal(s.attend(q=q, check=False), first)


# ---- together ----------------------------------------------------------------------------
def test_a_layer_in_graphs(hip):
    """The attention half of a layer as a batch goes through it: rows quantised, their product with the weights of queries, keys and
    values, into the cache, attention, and the product behind it; captured once and replayed while the sequences grow, beside the same calls
    without a graph on another stream and cache."""
    from instantllm_amd import mx
    heads, kv, dim, width, steps, seqs = 14, 2, 64, 896, 5, 6
    qkv = (heads + 2 * kv) * dim
    rng = np.random.default_rng(2)
    s = MxSetup(hip, [(20 * i + 1 + steps, 1) for i in range(seqs)], heads=heads, kv=kv, dim=dim, one_row=True, streams=2)
    lens = s.lens - steps
    w1, w2 = (M.quantize(rng.standard_normal((n, width)) * 0.03, "mxf4") for n in (qkv, width))
    d1, d2 = ([hip.put(a) for a in w] for w in (w1, w2))
    bias = hip.put(rng.standard_normal(qkv, dtype=np.float32))

    class Side:
        def __init__(self):
            self.k, self.v = hip.put(s.k_bits), hip.put(s.v_bits)
            self.lens = hip.put(lens)
            self.x, self.c, self.p = hip.alloc(2 * seqs * width), hip.alloc(seqs * width), hip.alloc(seqs * width // 32)
            self.y, self.q, self.o, self.out = hip.alloc(4 * seqs * qkv), hip.alloc(2 * seqs * width), hip.alloc(2 * seqs * width), hip.alloc(4 * seqs * width)
            self.batch = s.op.batch(self.lens, s.d_table, s.width, s.pages, seqs, table_stride=s.width + 2)

        def work(self, st):
            mx.quantize(self.x, self.c, self.p, seqs, width, stream=st)
            mx.product(self.c, self.p, *d1, self.y, seqs, qkv, width, dtype="f32", bias=bias, stream=st)
            s.op.append(self.batch, self.k, self.v, q=self.y, k=self.y + 4 * width, v=self.y + 4 * (width + kv * dim), q_out=self.q, x_dtype="f32", x_stride=qkv, stream=st)
            s.op.attend(self.batch, self.k, self.v, self.q, self.o, stream=st)
            mx.quantize(self.o, self.c, self.p, seqs, width, stream=st)
            mx.product(self.c, self.p, *d2, self.out, seqs, width, width, dtype="f32", stream=st)
    a, b = Side(), Side()
    s1, s2 = hip.stream(), hip.stream()
    graph = hip.capture(s1, lambda: a.work(s1))
    like = np.empty((seqs, width), np.float32)
    for i in range(steps):
        lens = lens + 1
        x = s.random_bits(seqs, width)
        for side in (a, b):
            hip.write(side.lens, lens)
            hip.write(side.x, x)
        hip.launch(graph, s1)
        b.work(s2)
        hip.sync()
        assert np.array_equal(hip.get(a.out, like), hip.get(b.out, like)) and np.array_equal(hip.get(a.k, s.k_bits), hip.get(b.k, s.k_bits))
        # and against the restatement, from what each call was given
        y = hip.get(b.y, np.empty((seqs, qkv), np.float32)).astype(np.float64).reshape(seqs, -1, dim)
        k, v = hip.get(b.k, s.k_bits), hip.get(b.v, s.v_bits)
        _, cached = O.append(s.geo, lens, s.table[:, :s.width], None, seqs, s.pages, y[:, :heads], y[:, heads:heads + kv], y[:, heads + kv:])
        for (p, t), (key, size, val) in cached.items():
            _between(s.parts(k)[0][p, :, t], s.parts(k)[1][p, :, t], key, 32 * U * size, "key")
            assert np.array_equal(s.parts(v)[0][p, :, t], M.quantize(val, "mxf8")[0])
        q, o = (O.from_bits(hip.get(d, np.empty((seqs, width), np.uint16)), "f16") for d in (b.q, b.o))
        ref, size, dots = O.attend(s.geo, lens, s.table[:, :s.width], None, seqs, s.pages, q.reshape(seqs, heads, dim), O.from_bits(s.view(k), "f16"),
                                   O.from_bits(s.view(v), "f16"), 0, 0, s.scale)
        for r in ref:
            tol = 2.0 ** -11 * (np.abs(ref[r]) + size[r]) + (2 * (dots[r] * (dim + 8) * U + 2.0 ** -21) + 300 * U) * size[r] + 2.0 ** -24
            assert (np.abs(o[r].reshape(heads, dim) - ref[r]) <= tol).all()
        c, w = M.values(*M.quantize(o, "mxf8"), "mxf8"), M.values(*w2, "mxf4")
        assert (np.abs(hip.get(b.out, like) - c @ w.T) <= (width + 2) * U * (np.abs(c) @ np.abs(w).T)).all()


def test_two_streams_and_a_graph_over_split_keys(hip):
    """Attention whose keys are split, on two streams at once and in a graph: each takes a workspace of its own."""
    s = MxSetup(hip, [(9000, 1), (7000, 1)], one_row=True, streams=3)
    s.upload()
    w = s.heads * s.dim
    qs = [s.random_bits(2, w) for _ in range(3)]
    want = [s.attend(q=q) for q in qs]
    s.op.release()
    dq, do = [hip.put(q) for q in qs], [hip.alloc(want[0].nbytes) for _ in qs]
    st = [hip.stream() for _ in range(3)]
    graph = hip.capture(st[2], lambda: s.op.attend(s.batch, s.kc, s.vc, dq[2], do[2], stream=st[2]))
    for _ in range(10):
        for p in do:
            hip.write(p, np.zeros_like(want[0]))
        hip.sync()
        for i in range(2):
            s.op.attend(s.batch, s.kc, s.vc, dq[i], do[i], stream=st[i])
        hip.launch(graph, st[2])
        hip.sync()
        for p, y in zip(do, want):
            assert np.array_equal(hip.get(p, y), y)
