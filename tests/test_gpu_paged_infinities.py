"""GPU tests of the paged-cache attention where rows see infinities and NaN among the values: an output is NaN, +inf or -inf
exactly where the definition says, wherever the value lies in its tile and however the keys are cut. A softmax weight is
positive, so a row that sees +inf (-inf) in a dim has +inf (-inf) there, and NaN if it sees both, or a NaN; the other dims are finite
and are held to the float64 restatement by the tolerances of test_gpu_paged.py."""
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


def check_kinds(s, got, window, sinks, out_dtype):
    """The kinds of all outputs, from the kinds of the values that their rows see (no weights in this)."""
    val = (O.from_bits(got, out_dtype) if out_dtype != "f32" else got.view(np.float32)).reshape(s.rows, s.heads, s.dim)
    v = O.from_bits(s.view(s.v_bits), s.dtype)
    kinds = np.stack([np.isposinf(v), np.isneginf(v), np.isnan(v)])   # [3][pages][slots][kv][dim]
    wild = 0
    for r, seq, p in O.rows_of(s.lens, s.row0, s.rows):
        seen = [O.slot(s.table[:, :s.width], s.pages, s.page, seq, j) for j in range(max(p + 1, 0)) if window == 0 or j > p - window or j < sinks]
        seen = [x for x in seen if x is not None]
        pg, sl = np.array(seen, int).reshape(-1, 2).T
        up, down, nan = np.repeat(kinds[:, pg, sl].any(1), s.heads // s.kv, axis=1)   # [heads][dim] each
        nan = nan | (up & down)
        want = np.where(nan, 3, np.where(up, 1, np.where(down, 2, 0)))
        g = val[r]
        have = np.where(np.isnan(g), 3, np.where(np.isposinf(g), 1, np.where(np.isneginf(g), 2, 0)))
        bad = want != have
        assert not bad.any(), (f"row {r} at {p}", np.argwhere(bad)[:4], "want, have (1 inf, 2 -inf, 3 nan)", want[bad][:4], have[bad][:4])
        wild += int((want > 0).sum())
    return wild


def put(s, seq, t, head, dims):
    """dims: {dim: value} of the value at position t of a sequence."""
    pg, sl = O.slot(s.table[:, :s.width], s.pages, s.page, seq, t)
    for d, x in dims.items():
        s.view(s.v_bits)[pg, sl, head, d] = O.to_bits(np.array([x], np.float32), s.dtype)[0]


def attend(s, window=0, sinks=0, out_dtype=None, **kw):
    with np.errstate(invalid="ignore", over="ignore"):   # (the restatement's own comparison of infinities)
        got = s.attend(window=window, sinks=sinks, out_dtype=out_dtype, **kw)
    return check_kinds(s, got, window, sinks, out_dtype or s.dtype)


INF, NAN = np.inf, np.nan
SHAPES = [(1, 6, 2), (3, 6, 2), (40, 6, 2), (150, 112, 112)]


@pytest.mark.parametrize("out_dtype", [None, "f32"], ids=["narrow", "f32"])
@pytest.mark.parametrize("dim,dtype", [(64, "f16"), (128, "f16"), (64, "bf16"), (128, "bf16")])
@pytest.mark.parametrize("rows,heads,kv", SHAPES, ids=["1", "3", "40", "150-prompt-kernel"])
def test_infinities_that_every_row_sees(hip, rows, heads, kv, dim, dtype, out_dtype):
    """In tiles that are seen whole, in the last one, and in several tiles of one dim."""
    s = Setup(hip, [(300, rows), (260, min(rows, 60)), (16, 1)], heads=heads, kv=kv, dim=dim, dtype=dtype)
    for t in (5, 70, 140):   # (all rows of the first sequence are behind position 149)
        put(s, 0, t, 0, {1: INF, 2: -INF, 40: INF})
    put(s, 0, 20, 0, {3: INF, 4: -INF, 5: INF})
    put(s, 0, 100, 0, {3: INF, 4: -INF, 5: -INF, 6: NAN})
    put(s, 0, 149, 1, {0: INF, dim - 1: -INF})
    put(s, 0, 299, 0, {7: INF, 2: INF})        # seen by the last row alone: -inf and +inf make NaN
    put(s, 1, 9, 1, {11: -INF, 12: NAN})
    put(s, 2, 15, 0, {13: INF})
    assert attend(s, out_dtype=out_dtype) > 0
    assert attend(s, window=250, sinks=7, out_dtype=out_dtype) > 0
    assert attend(s, window=30, sinks=6, out_dtype=out_dtype) > 0


@pytest.mark.parametrize("out_dtype", [None, "f32"], ids=["narrow", "f32"])
@pytest.mark.parametrize("dim,dtype", [(64, "f16"), (128, "bf16")])
@pytest.mark.parametrize("seqs,heads,kv", [([(9000, 1)], 4, 2), ([(9000, 20)], 4, 1), ([(6000, 40)] + [(100 + i, 40) for i in range(7)], 64, 32)],
                         ids=["1", "20", "both"])
def test_infinities_with_weights_of_next_to_nothing(hip, seqs, heads, kv, dim, dtype, out_dtype):
    """A few keys' scores lie 110 to 400 above the others', whose weights underflow in float32: the infinities among the others' values
    reach the rows all the same, from tiles before and behind those keys, and from other parts of the keys. (Up to 700 the float64
    restatement's weights do not underflow.)"""
    s = Setup(hip, seqs, heads=heads, kv=kv, dim=dim, dtype=dtype)
    w = s.heads * s.dim
    q = s.rng.standard_normal((s.rows, w), dtype=np.float32)
    q[:, ::dim] = 30.0                       # dim 0 of every head
    keys = s.view(s.k_bits)
    scale = 30 * s.scale
    keys[..., 0] = 0
    for t, score in ((3000, 110.0), (3001, 250.0), (5200, 400.0)):
        pg, sl = O.slot(s.table, s.pages, s.page, 0, t)
        keys[pg, sl, :, 0] = O.to_bits(np.array([score / scale], np.float32), dtype)[0]
    put(s, 0, 17, 0, {1: INF, 2: -INF, 3: INF})
    put(s, 0, 2990, 0, {4: INF, 3: -INF})
    put(s, 0, 3064, 0, {5: -INF})
    put(s, 0, 5000, kv - 1, {6: INF, 7: NAN})
    put(s, 0, 5900, 0, {8: -INF, 9: INF})
    if seqs[0][0] > 8000:
        put(s, 0, 8000, 0, {10: INF, 1: -INF})
    assert attend(s, out_dtype=out_dtype, q=O.to_bits(q, dtype)) > 0


@pytest.mark.parametrize("rows,heads,kv", [(1, 4, 2), (150, 112, 112)], ids=["step", "prompt-kernel"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_rows_whose_scores_are_all_minus_infinity_are_zeros(hip, rows, heads, kv, dtype):
    """Whatever the values are; and NaN scores make all of a row NaN."""
    s = Setup(hip, [(300, rows)], heads=heads, kv=kv, dtype=dtype)
    s.view(s.k_bits)[..., 0] = O.to_bits(np.array([-INF], np.float32), dtype)[0]
    put(s, 0, 5, 0, {1: INF, 2: NAN})
    put(s, 0, 299, 1, {1: INF, 2: NAN})
    q = np.abs(s.rng.standard_normal((s.rows, heads * 64), dtype=np.float32)) + 0.5
    for out_dtype in (s.dtype, "f32"):
        got = s.attend(q=O.to_bits(q, dtype), out_dtype=out_dtype, check=False)
        assert not got.any()
    s.kc = None
    pg, sl = O.slot(s.table, s.pages, s.page, 0, 8)
    s.view(s.k_bits)[pg, sl, 0, 0] = O.to_bits(np.array([NAN], np.float32), dtype)[0]
    got = s.attend(q=O.to_bits(q, dtype), out_dtype="f32", check=False).view(np.float32).reshape(s.rows, heads, 64)
    assert np.isnan(got[:, :heads // kv]).all()
    assert not got[:, heads // kv:].any()


@pytest.mark.parametrize("rows,heads,kv", [(1, 4, 2), (40, 4, 2), (150, 112, 112)], ids=["step", "40", "prompt-kernel"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_infinite_scores_and_queries_stay_in_their_rows(hip, rows, heads, kv, dtype):
    """A key with +inf, and queries with infinities and NaN, make whole rows NaN, and no other row."""
    s = Setup(hip, [(300, rows), (200, 1)], heads=heads, kv=kv, dtype=dtype)
    q = np.abs(s.rng.standard_normal((s.rows, heads, 64), dtype=np.float32)) + 0.5
    plain = {t: s.attend(q=O.to_bits(q.reshape(s.rows, -1), dtype), out_dtype=t) for t in (dtype, "f32")}
    wild = q.copy()
    wild[0, 0, 3], wild[-1, -1, 5] = NAN, INF
    v = s.view(s.k_bits)
    seen = [O.slot(s.table[:, :s.width], s.pages, s.page, 0, t) for t in range(300)]
    assert all((O.from_bits(v[p, t, 0, 5], dtype) != 0).all() for p, t in seen)
    for t, before in plain.items():
        got = s.attend(q=O.to_bits(wild.reshape(s.rows, -1), dtype), out_dtype=t, check=False).reshape(s.rows, heads, 64)
        val = got.view(np.float32) if t == "f32" else O.from_bits(got, t)
        want = before.reshape(got.shape)
        for r in range(s.rows):
            for h in range(heads):
                if (r, h) in ((0, 0), (s.rows - 1, heads - 1)):
                    assert np.isnan(val[r, h]).all(), (r, h)
                else:
                    assert np.array_equal(got[r, h], want[r, h]), (r, h)
    pg, sl = seen[70]
    v[pg, sl, 0, 9] = O.to_bits(np.array([INF], np.float32), dtype)[0]
    s.kc = None
    for t, before in plain.items():
        got = s.attend(q=O.to_bits(q.reshape(s.rows, -1), dtype), out_dtype=t, check=False).reshape(s.rows, heads, 64)
        val, want, group = got.view(np.float32) if t == "f32" else O.from_bits(got, t), before.reshape(got.shape), heads // kv
        assert np.isnan(val[:rows, :group]).all()
        assert np.array_equal(got[:rows, group:], want[:rows, group:]) and np.array_equal(got[rows:], want[rows:])


@pytest.mark.parametrize("length,rows,heads,kv", [(9000, 1, 4, 2), (400, 150, 112, 112)], ids=["step", "prompt-kernel"])
def test_graphs_follow_values_that_become_infinite(hip, length, rows, heads, kv):
    """One graph over finite values, over infinities and over finite ones again."""
    s = Setup(hip, [(length, rows), (200, rows)], heads=heads, kv=kv)
    s.upload()
    clean, w = s.v_bits.copy(), heads * 64
    q = s.random_bits(s.rows, w)
    put(s, 0, 100, 0, {1: INF, 2: -INF})
    put(s, 1, 20, 1, {3: NAN})
    dirty = s.v_bits.copy()
    st = hip.stream()
    dq, do = hip.put(q), hip.alloc(2 * s.rows * w)
    graph = hip.capture(st, lambda: s.op.attend(s.batch, s.kc, s.vc, dq, do, stream=st))
    for turn in range(5):
        s.v_bits[...] = dirty if turn % 2 else clean
        hip.write(s.vc, s.v_bits)
        with np.errstate(invalid="ignore"):
            want = s.attend(q=q, check=turn < 2)
        hip.write(do, np.zeros_like(want))
        hip.sync()
        for _ in range(2):
            hip.launch(graph, st)
        got = hip.get(do, want)
        assert np.array_equal(got, want), turn
        assert (check_kinds(s, got, 0, 0, "f16") > 0) == (turn % 2 == 1)
