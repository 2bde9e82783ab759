"""Float64 restatement of the paged-cache operators: new rows into the cache, and their attention
over it, position by position as include/ill_hip.h defines them. Types: "f32", "f16", "bf16"; 16-bit
arrays are held as uint16 bits."""
from __future__ import annotations

import numpy as np

HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
LEAST = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}   # smallest subnormal


def to_bits(x: np.ndarray, dtype: str) -> np.ndarray:
    """Rounded to nearest, ties to even."""
    x = np.ascontiguousarray(x, np.float32)
    if dtype == "f32":
        return x
    if dtype == "f16":
        return x.astype(np.float16).view(np.uint16)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bits(b: np.ndarray, dtype: str) -> np.ndarray:
    if dtype == "f32":
        return b.astype(np.float64)
    if dtype == "f16":
        return b.view(np.float16).astype(np.float64)
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def rows_of(lens, row0, rows):
    """(row, sequence, position) of every new row; row0 None: row s is sequence s's only one."""
    out = []
    for s, n in enumerate(lens):
        a, b = (s, s + 1) if row0 is None else (row0[s], row0[s + 1])
        out += [(r, s, max(int(n), 0) - (b - r)) for r in range(a, min(b, rows))]
    return out


def slot(table, pages, page_size, s, t):
    """(page, slot) of position t of sequence s; None where there is no such place."""
    if t < 0 or t >= table.shape[1] * page_size:
        return None
    page = int(table[s, t // page_size])
    return (page, t % page_size) if 0 <= page < pages else None


def turn(x, position, rotary_dim, base, interleaved):
    """x [..., dim] rotated; also the size of what went into each output."""
    y, size = x.copy(), np.abs(x)
    if rotary_dim:
        i = np.arange(rotary_dim // 2)
        angle = position * base ** (-2.0 * i / rotary_dim)
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rotary_dim // 2)
        c, s = np.cos(angle), np.sin(angle)
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
        size[..., a] = size[..., b] = np.abs(x[..., a]) + np.abs(x[..., b])
    return y, size


def append(geo, lens, table, row0, rows, pages, q, k, v, bias=None, q_norm=None, k_norm=None, positions=None):
    """geo: heads, kv_heads, head_dim, page_size, rotary_dim, rope_base, interleaved, norm_eps. q, k, v: float64 [rows][heads][dim].
    Returns ({row: (query, size)}, {(page, slot): (key, key size, value)}): what has to be there, and the magnitudes that rounding
    errors in float32 are relative to."""
    heads, kv, dim = geo["heads"], geo["kv_heads"], geo["head_dim"]
    queries, cached = {}, {}
    for r, s, t in rows_of(lens, row0, rows):
        parts = [q[r].copy(), k[r].copy(), v[r].copy()]
        if bias is not None:
            b = bias.reshape(-1, dim)
            parts = [p + c for p, c in zip(parts, (b[:heads], b[heads:heads + kv], b[heads + kv:]))]
        for i, gamma in enumerate((q_norm, k_norm)):
            if gamma is not None:
                parts[i] = parts[i] / np.sqrt((parts[i] ** 2).mean(-1, keepdims=True) + geo["norm_eps"]) * gamma
        at = t if positions is None else int(positions[r])
        turned = [turn(p, at, geo["rotary_dim"], geo["rope_base"], geo["interleaved"]) for p in parts[:2]]
        queries[r] = turned[0]
        place = slot(table, pages, geo["page_size"], s, t)
        if place is not None:
            cached[place] = (*turned[1], parts[2])
    return queries, cached


def attend(geo, lens, table, row0, rows, pages, q, k_cache, v_cache, window, sinks, scale):
    """k_cache, v_cache: float64 [pages][page_size][kv_heads][dim]. Returns ({row: output}, {row: sum of the weighted values' sizes},
    {row: a bound of sum |q k| scale over the keys seen})."""
    heads, kv, dim = geo["heads"], geo["kv_heads"], geo["head_dim"]
    out, size, dots = {}, {}, {}
    for r, s, p in rows_of(lens, row0, rows):
        places = [slot(table, pages, geo["page_size"], s, j) for j in range(max(p + 1, 0))
                  if window == 0 or j > p - window or j < sinks]
        places = [x for x in places if x is not None]
        o, z, d = np.zeros((heads, dim)), np.zeros((heads, dim)), np.zeros((heads, 1))
        if places:
            pg, sl = np.array(places).T
            for h in range(heads):
                key, val = k_cache[pg, sl, h * kv // heads], v_cache[pg, sl, h * kv // heads]
                score = key @ q[r, h] * scale
                w = np.exp(score - score.max())
                w /= w.sum()
                o[h], z[h] = w @ val, w @ np.abs(val)
                d[h] = (np.abs(key) @ np.abs(q[r, h])).max() * scale
        out[r], size[r], dots[r] = o, z, d
    return out, size, dots
