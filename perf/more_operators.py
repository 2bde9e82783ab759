"""Cases that measure the microscaled operators: `instantllm_amd.mx` and the caches of `instantllm_amd.paged.PagedAttention` with
`cache="mxf8"`.

A microscaled row is blocks of 32 values that share a power of two: a byte e stands for 2^(e - 127), 255 for a block of NaN. Codes
are e4m3 ("mxf8", a byte) or e2m1 ("mxf4", two to a byte, the first in the low four bits). A block's power is floor(log2 of its
largest size) - 8 (mxf4: - 2), never below 2^-127, its values divided by it are rounded to nearest, ties to even, and end at
+-448 (+-6).

  quantize  rows to microscaled ones, and back to values (quantize, dequantize)
  linear    a layer's product: rows quantised, times a matrix of mxf4 rows, plus a bias (quantize, product)
  append    new rows into a cache of mxf8 keys and values, and what then stands there (append, read)
  read      whole sequences' keys and values out of such a cache
  attend    attention over such a cache

A page of the cache holds [kv heads][page size][head size] codes and, behind them, [kv heads][page size][head size / 32] powers.
Head layouts are (query heads, key/value heads, head size): (14, 2, 64) is the model that the engine serves.
"""
import functools
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LAYOUTS = [(14, 2, 64), (32, 8, 128), (12, 12, 64), (16, 1, 128), (28, 4, 128)]
BASE, EPS = 1e6, 1e-6
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def listed():
    return [
        # one row of the engine's hidden size, and the widest activations of its longest prompt chunk
        {"name": "quantize_step", "kind": "quantize", "rows": 1, "cols": 896, "x": "f16", "format": "mxf8"},
        {"name": "quantize_chunk4096", "kind": "quantize", "rows": 4096, "cols": 4864, "x": "bf16", "format": "mxf4"},
        # one row's queries, keys and values (float32 out, as the cache's rows may come)
        {"name": "linear_step", "kind": "linear", "rows": 1, "cols": 1152, "inner": 896, "x": "f16", "format": "mxf8", "out": "f32", "bias": True},
        # the vocabulary for a batch of 16
        {"name": "linear_vocab16", "kind": "linear", "rows": 16, "cols": 151936, "inner": 896, "x": "bf16", "format": "mxf8", "out": "bf16", "bias": False},
        # large products of prompts: the way down of the engine's model for a ragged batch, and a square one
        {"name": "linear_prompts5001", "kind": "linear", "rows": 5001, "cols": 896, "inner": 4864, "x": "f16", "format": "mxf8", "out": "f16", "bias": False},
        {"name": "linear_8192", "kind": "linear", "rows": 8192, "cols": 8192, "inner": 8192, "x": "bf16", "format": "mxf4", "out": "bf16", "bias": False},
        # new rows: a decode step of 64 requests with head norms, the engine's longest prompt chunk
        {"name": "append_batch64", "kind": "append", "heads": 32, "kv": 8, "dim": 128, "type": "bf16", "x": "bf16", "page": 32,
         "seqs": 64, "rows": 1, "lo": 2, "hi": 700, "bias": False, "norm": True, "mix": 2},
        {"name": "append_chunk4096", "kind": "append", "heads": 14, "kv": 2, "dim": 64, "type": "f16", "x": "f32", "page": 64,
         "seqs": 1, "rows": 4096, "lo": 8200, "hi": 8200, "bias": True, "norm": False, "mix": 3},
        # a prefix that moves to another cache
        {"name": "read_ragged30", "kind": "read", "heads": 32, "kv": 8, "dim": 128, "type": "bf16", "out": "bf16", "page": 16,
         "seqs": 30, "rows": 9000, "lo": 100, "hi": 9000, "mix": 4},
        # decode steps: a batch with contexts of very different lengths, one very long request
        {"name": "step_64_ragged", "kind": "attend", "heads": 32, "kv": 8, "dim": 128, "type": "bf16", "out": "bf16", "page": 16,
         "seqs": 64, "rows": 1, "lo": 100, "hi": 9000, "window": 0, "sinks": 0, "mix": 7},
        {"name": "step_1x131071", "kind": "attend", "heads": 14, "kv": 2, "dim": 64, "type": "f16", "out": "f32", "page": 64,
         "seqs": 1, "rows": 1, "lo": 131071, "hi": 131071, "window": 0, "sinks": 0, "mix": 6},
        # a mixed batch: prompts' chunks beside single tokens
        {"name": "prompt_mixed9", "kind": "attend", "heads": 32, "kv": 8, "dim": 128, "type": "bf16", "out": "bf16", "page": 16,
         "seqs": 9, "rows": 700, "lo": 400, "hi": 5000, "window": 0, "sinks": 0, "mix": 11},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    what = rng.choice(["quantize", "linear", "linear", "linear", "append", "read", "step", "step", "prompt"])
    if what == "quantize":
        cols = 32 * _log_int(rng, 1, 300)
        return {"kind": "quantize", "rows": _log_int(rng, 1, min(200000, 20000000 // cols)), "cols": cols, "x": rng.choice(["f32", "f16", "bf16"]),
                "format": rng.choice(["mxf8", "mxf4"])}
    if what == "linear":
        inner = 32 * rng.choice([_log_int(rng, 1, 256), 4 * _log_int(rng, 1, 64)])
        cols = _log_int(rng, 17, min(160000, 140000000 // inner))
        return {"kind": "linear", "rows": _log_int(rng, 1, min(8192, 60000000 // cols)), "cols": cols, "inner": inner, "x": rng.choice(["f32", "f16", "bf16"]),
                "format": rng.choice(["mxf8", "mxf4"]), "out": rng.choice(["f32", "f16", "bf16"]), "bias": rng.random() < 0.5}
    heads, kv, dim = rng.choice(LAYOUTS)
    case = {"heads": heads, "kv": kv, "dim": dim, "type": rng.choice(["f16", "bf16"]), "page": rng.choice([16, 32, 64, 128, 256]),
            "mix": rng.randrange(1 << 20)}
    if what == "append":
        seqs = _log_int(rng, 1, 64)
        rows = rng.choice([1, _log_int(rng, 2, 12000 // seqs)])
        lo = rows + rng.randint(0, 300)
        return {**case, "kind": "append", "x": rng.choice(["f32", case["type"]]), "seqs": seqs, "rows": rows, "lo": lo,
                "hi": lo + _log_int(rng, 1, 500), "bias": rng.random() < 0.5, "norm": rng.random() < 0.5}
    if what == "read":
        seqs = _log_int(rng, 1, 30)
        hi = _log_int(rng, 1, 60000 // seqs)
        return {**case, "kind": "read", "out": rng.choice(["f32", case["type"]]), "seqs": seqs, "rows": hi, "lo": max(1, hi // rng.choice([1, 4, 40])), "hi": hi}
    window = rng.choice([0, 0, _log_int(rng, 16, 4096)])
    case.update(kind="attend", out=rng.choice([case["type"], case["type"], "f32"]), window=window,
                sinks=rng.choice([0, rng.randint(1, 40)]) if window else 0)
    if what == "step":
        seqs = _log_int(rng, 1, 200)
        hi = _log_int(rng, 1, min(131071, 400000 // seqs))
        return {**case, "seqs": seqs, "rows": 1, "lo": max(1, hi // rng.choice([1, 4, 40])), "hi": hi}
    seqs = rng.randint(1, 9)
    rows = _log_int(rng, 2, 6000 // seqs)
    hi = rows + _log_int(rng, 1, 2000)
    return {**case, "seqs": seqs, "rows": rows, "lo": rng.choice([rows, hi]), "hi": hi}


def _shape(case):
    """(lengths, new rows) of the sequences: the first one is the longest, every third one of a batch of prompts has a single
    new row, the others any number up to `rows`; all of its positions where a cache is read. They belong to the case, not to the
    inputs' seed."""
    rng = random.Random(case["mix"])
    lens = [case["hi"]] + [_log_int(rng, case["lo"], case["hi"]) for _ in range(case["seqs"] - 1)]
    if case["kind"] == "read":
        return lens, lens
    rows = [min(n, case["rows"] if i == 0 or case["rows"] == 1 else 1 if i % 3 == 2 else rng.randint(1, case["rows"]))
            for i, n in enumerate(lens)]
    return lens, rows


def _tables(case, seed):
    """Page table of random distinct pages (pages past a sequence's last are -1), and the number of pages."""
    lens, _ = _shape(case)
    need = [-(-n // case["page"]) for n in lens]
    pages = sum(need) + 3
    order = random.Random(seed).sample(range(pages), sum(need))
    table = torch.full((case["seqs"], max(need)), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    return table, pages


@functools.lru_cache(maxsize=None)
def _handle(heads, kv, dim, page, dtype):
    """The one handle that a program keeps for a model."""
    from instantllm_amd.paged import PagedAttention
    return PagedAttention(heads, kv, dim, page_size=page, dtype=dtype, cache="mxf8", rope_base=BASE, norm_eps=EPS)


# ---- microscaled rows in elementary operations ---------------------------------------------
def _two_to(e):
    """2^e in float64, from its bits: e integers, -1022 to 1023."""
    return (e.long() + 1023 << 52).view(torch.float64)


def _to_mx(x, fmt):
    """Codes and powers of the float32 blocks of 32 along the last axis."""
    x = x.unflatten(-1, (-1, 32))
    top, least, most = (8, 2.0 ** -6, 448.0) if fmt == "mxf8" else (2, 1.0, 6.0)
    size = x.abs().amax(-1)
    power = (torch.frexp(size).exponent.clamp(min=-300) - 1 - top).clamp(min=-127)   # (the exponent of 0 says nothing: any power will do)
    power = torch.where(size == 0, -127, power)
    y = (x * _two_to(-power[..., None])).clamp(-most, most)
    step = _two_to(torch.frexp(y.abs().clamp(min=least)).exponent - (4 if fmt == "mxf8" else 2))
    y = torch.round(y / step) * step
    y = torch.where((y == 0) & torch.signbit(x), -0.0, y).float()
    if fmt == "mxf8":
        codes = y.to(torch.float8_e4m3fn).view(torch.uint8).flatten(-2)
    else:
        codes = torch.searchsorted(torch.tensor(E2M1, device=x.device), y.abs().contiguous()).to(torch.uint8) | (torch.signbit(y).to(torch.uint8) << 3)
        codes = codes.flatten(-2)
        codes = codes[..., ::2] | codes[..., 1::2] << 4
    return codes, (power + 127).to(torch.uint8)


def _from_mx(codes, powers, fmt):
    if fmt == "mxf8":
        y = codes.view(torch.float8_e4m3fn).float()
    else:
        values = torch.tensor(E2M1 + [-v for v in E2M1], device=codes.device)
        y = values[torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()]
    return (y.unflatten(-1, (-1, 32)) * _two_to(powers[..., None].int() - 127).float()).flatten(-2)


def _in_parts(f, x, *more):
    """f of a matrix's rows, few enough at a time for the memory that its steps take."""
    n = max(1, (1 << 25) // x.shape[-1])
    parts = [f(p, *more) for p in x.split(n)]
    return tuple(torch.cat(p) for p in zip(*parts))


def _values_of_cache(cache, case):
    """[pages][kv heads][page size][head size] values of a cache."""
    kv, page, dim = case["kv"], case["page"], case["dim"]
    n = kv * page * dim
    return _from_mx(cache[:, :n].reshape(-1, kv, page, dim), cache[:, n:].reshape(-1, kv, page, dim // 32), "mxf8")


def _spread(normal, *shape):
    """Activations: sizes differ between rows, and a few columns are much larger."""
    x = normal(*shape) * torch.exp(normal(shape[0], 1))
    x[:, ::61] *= 8
    return x


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    if case["kind"] in ("quantize", "linear"):
        rows, cols = case["rows"], case["cols"] if case["kind"] == "quantize" else case["inner"]
        state = {"case": case, "x": _spread(normal, rows, cols).to(DTYPES[case["x"]]),
                 "codes": torch.empty(rows, cols if case["format"] == "mxf8" else cols // 2, dtype=torch.uint8, device="cuda"),
                 "powers": torch.empty(rows, cols // 32, dtype=torch.uint8, device="cuda")}
        if case["kind"] == "quantize":
            return {**state, "y": torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")}
        n = case["cols"]
        w, wp = _in_parts(_to_mx, normal(n, cols) * 0.02, "mxf4")
        return {**state, "w": w, "wp": wp, "bias": normal(n) if case["bias"] else None, "y": torch.empty(rows, n, dtype=DTYPES[case["out"]], device="cuda")}
    heads, kv, dim, page, dt = case["heads"], case["kv"], case["dim"], case["page"], DTYPES[case["type"]]
    lens, rows = _shape(case)
    table, pages = _tables(case, seed)

    def cache():
        codes, powers = _in_parts(_to_mx, normal(pages * kv * page, dim), "mxf8")
        return torch.cat((codes.view(pages, -1), powers.view(pages, -1)), 1)

    total = sum(rows)
    state = {"case": case, "k_cache": cache(), "v_cache": cache(), "lens": torch.tensor(lens, dtype=torch.int32).cuda(), "table": table.cuda(), "pages": pages,
             "row0": torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], dtype=torch.int32).cuda(), "total": total, "most": max(rows),
             "handle": _handle(heads, kv, dim, page, case["type"]) if own else None}
    if case["kind"] != "attend":
        out = DTYPES[case.get("out", case["type"])]
        state.update(k=torch.empty(total, kv * dim, dtype=out, device="cuda"), v=torch.empty(total, kv * dim, dtype=out, device="cuda"))
    if case["kind"] == "append":
        state.update(x=normal(total, (heads + 2 * kv) * dim).to(DTYPES[case["x"]]), q=torch.empty(total, heads * dim, dtype=dt, device="cuda"),
                     bias=normal((heads + 2 * kv) * dim) if case["bias"] else None,
                     q_norm=1 + 0.2 * normal(dim) if case["norm"] else None, k_norm=1 + 0.2 * normal(dim) if case["norm"] else None)
    elif case["kind"] == "attend":   # some queries' scores are nearly even, others' fall on a few keys
        state.update(q=(normal(total, heads, dim) * (0.5 + 3 * torch.rand(total, heads, 1, generator=gen, device="cuda"))).to(dt).view(total, -1),
                     out=torch.empty(total, heads * dim, dtype=DTYPES[case["out"]], device="cuda"))
    return state


# ---- the plain forms -----------------------------------------------------------------------
def _plain_quantize(state):
    fmt = state["case"]["format"]
    state["codes"], state["powers"] = _to_mx(state["x"].float(), fmt)
    state["y"].copy_(_from_mx(state["codes"], state["powers"], fmt))
    return {"values": state["y"]}


def _plain_linear(state):
    fmt = state["case"]["format"]
    x = _from_mx(*_to_mx(state["x"].float(), fmt), fmt)
    y = x @ _from_mx(state["w"], state["wp"], "mxf4").T
    if state["bias"] is not None:
        y = y + state["bias"]
    state["y"].copy_(y)
    return {"y": state["y"]}


def _places(state):
    """Each new row's sequence and position."""
    counts = state["row0"][1:] - state["row0"][:-1]
    seq = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), counts.long(), output_size=state["total"])
    at = torch.arange(state["total"], device="cuda") - state["row0"][seq]
    return seq, at, state["lens"][seq] - counts[seq] + at


def _slots(state):
    """Each new row's page and slot."""
    seq, _, pos = _places(state)
    page = state["case"]["page"]
    return state["table"][seq, torch.div(pos, page, rounding_mode="floor")].long(), pos.long() % page


def _plain_read(state):
    case = state["case"]
    kv, page, dim = case["kv"], case["page"], case["dim"]
    where, slot = _slots(state)
    n = kv * page * dim
    for cache, out in ((state["k_cache"], state["k"]), (state["v_cache"], state["v"])):
        codes, powers = cache[:, :n].reshape(-1, kv, page, dim), cache[:, n:].reshape(-1, kv, page, dim // 32)
        out.copy_(_from_mx(codes[where, :, slot], powers[where, :, slot], "mxf8").flatten(1))
    return {"k": state["k"], "v": state["v"]}


def _plain_append(state):
    case = state["case"]
    heads, kv, dim, page = case["heads"], case["kv"], case["dim"], case["page"]
    _, _, pos = _places(state)
    x = state["x"].float()
    if case["bias"]:
        x = x + state["bias"]
    x = x.view(-1, heads + 2 * kv, dim)
    q, k, v = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
    if case["norm"]:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + EPS) * state["q_norm"]
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + EPS) * state["k_norm"]
    angle = pos.double()[:, None, None] * BASE ** (-torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim)
    cos, sin = angle.cos().float(), angle.sin().float()

    def turn(t):
        a, b = t[..., :dim // 2], t[..., dim // 2:]
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

    where, slot = _slots(state)
    n = kv * page * dim
    for cache, rows in ((state["k_cache"], turn(k)), (state["v_cache"], v)):
        codes, powers = _to_mx(rows, "mxf8")
        cache[:, :n].unflatten(1, (kv, page, dim))[where, :, slot] = codes
        cache[:, n:].unflatten(1, (kv, page, dim // 32))[where, :, slot] = powers
    state["q"].copy_(turn(q).view(-1, heads * dim))
    return {"q": state["q"], **_plain_read(state)}


def _plain_attend(state):
    """All sequences at once, padded to the longest one and to the most rows."""
    case = state["case"]
    heads, kv, dim, page = case["heads"], case["kv"], case["dim"], case["page"]
    group, most = heads // kv, state["most"]
    seq, at, pos = _places(state)
    seqs, longest = case["seqs"], state["table"].shape[1] * page
    rows = torch.zeros(seqs, most, heads, dim, device="cuda")
    rows[seq, at] = state["q"].view(-1, heads, dim).float()
    place = torch.full((seqs, most), -1, device="cuda")
    place[seq, at] = pos.long()
    pick = state["table"].clamp(min=0).long()
    k, v = (_values_of_cache(c, case)[pick].transpose(1, 2).reshape(seqs, kv, longest, dim) for c in (state["k_cache"], state["v_cache"]))
    rows = rows.view(seqs, most, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv, group * most, dim)
    key = torch.arange(longest, device="cuda")
    seen = key <= place[..., None]
    if case["window"]:
        seen = seen & ((key > place[..., None] - case["window"]) | (key < case["sinks"]))
    seen = seen[:, None].repeat(1, 1, group, 1)
    scores = (rows @ k.transpose(2, 3).contiguous()) / math.sqrt(dim)
    scores = scores.masked_fill(~seen, float("-inf"))
    weight = (scores - scores.amax(-1, keepdim=True).clamp(min=-3e38)).exp()
    total = weight.sum(-1, keepdim=True)
    out = (weight @ v) / total.clamp(min=1e-38)
    out = out.view(seqs, kv, group, most, dim).permute(0, 3, 1, 2, 4).reshape(seqs, most, heads * dim)
    state["out"].copy_(out[seq, at])
    return {"out": state["out"]}


# ---- the framework's calls -----------------------------------------------------------------
def _own_quantize(state):
    from instantllm_amd import mx
    case = state["case"]
    codes, powers = state["codes"].data_ptr(), state["powers"].data_ptr()
    mx.quantize(state["x"].data_ptr(), codes, powers, case["rows"], case["cols"], format=case["format"], dtype=case["x"])
    mx.dequantize(codes, powers, state["y"].data_ptr(), case["rows"], case["cols"], format=case["format"], dtype="bf16")
    return {"values": state["y"]}


def _own_linear(state):
    from instantllm_amd import mx
    case = state["case"]
    codes, powers = state["codes"].data_ptr(), state["powers"].data_ptr()
    mx.quantize(state["x"].data_ptr(), codes, powers, case["rows"], case["inner"], format=case["format"], dtype=case["x"])
    mx.product(codes, powers, state["w"].data_ptr(), state["wp"].data_ptr(), state["y"].data_ptr(), case["rows"], case["cols"], case["inner"],
               format=case["format"], dtype=case["out"], bias=None if state["bias"] is None else state["bias"].data_ptr())
    return {"y": state["y"]}


def _batch(state):
    """The batch as the calls take it: device addresses and sizes."""
    return state["handle"].batch(lens=state["lens"].data_ptr(), table=state["table"].data_ptr(), table_width=state["table"].shape[1],
                                 pages=state["pages"], seqs=state["case"]["seqs"], rows=state["total"], row0=state["row0"].data_ptr(),
                                 max_rows=state["most"])


def _own_read(state):
    case = state["case"]
    state["handle"].read(_batch(state), state["k_cache"].data_ptr(), state["v_cache"].data_ptr(), state["k"].data_ptr(), state["v"].data_ptr(),
                         dtype=case.get("out", case["type"]))
    return {"k": state["k"], "v": state["v"]}


def _own_append(state):
    case = state["case"]
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    x, size, width = state["x"], state["x"].element_size(), (heads + 2 * kv) * dim
    address = x.data_ptr()
    state["handle"].append(_batch(state), state["k_cache"].data_ptr(), state["v_cache"].data_ptr(), q=address, k=address + heads * dim * size,
                           v=address + (heads + kv) * dim * size, q_out=state["q"].data_ptr(), x_dtype=case["x"], x_stride=width,
                           bias=state["bias"].data_ptr() if case["bias"] else None, q_norm=state["q_norm"].data_ptr() if case["norm"] else None,
                           k_norm=state["k_norm"].data_ptr() if case["norm"] else None)
    return {"q": state["q"], **_own_read(state)}


def _own_attend(state):
    case = state["case"]
    state["handle"].attend(_batch(state), state["k_cache"].data_ptr(), state["v_cache"].data_ptr(), state["q"].data_ptr(),
                           state["out"].data_ptr(), out_dtype=case["out"], window=case["window"], sinks=case["sinks"])
    return {"out": state["out"]}


_PLAIN = {"quantize": _plain_quantize, "linear": _plain_linear, "append": _plain_append, "read": _plain_read, "attend": _plain_attend}
_OWN = {"quantize": _own_quantize, "linear": _own_linear, "append": _own_append, "read": _own_read, "attend": _own_attend}


@torch.no_grad()
def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["kind"]](state)


# ---- what a pass needs, and what it is in 64 bits -------------------------------------------
def _visible(case, p):
    """How many positions the row at position p sees."""
    if not case["window"] or p < case["window"]:
        return p + 1
    return case["window"] + min(case["sinks"], p + 1 - case["window"])


def _pairs(case, first, n):
    """The sum of _visible over the positions first .. first + n - 1."""
    return sum(_visible(case, p) for p in range(first, first + n))


def _distinct(case, first, n):
    """How many positions some row of first .. first + n - 1 sees."""
    end = first + n
    if not case["window"]:
        return end
    low = max(0, first - case["window"] + 1)
    return end - low + min(case["sinks"], low)


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["kind"] == "quantize":
        n = case["rows"] * case["cols"]
        return {"bytes": float(n * (size[case["x"]] + 2)), "flops": float(4 * n)}
    if case["kind"] == "linear":
        rows, cols, inner = case["rows"], case["cols"], case["inner"]
        return {"bytes": rows * inner * size[case["x"]] + cols * inner * (0.5 + 1 / 32) + rows * cols * size[case["out"]] + 4.0 * cols * case["bias"],
                "flops": 2.0 * rows * cols * inner}
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    lens, rows = _shape(case)
    total = sum(rows)
    tables = 4 * (2 * case["seqs"] + 1 + sum(-(-n // case["page"]) for n in lens))
    held = dim + dim // 32   # bytes of a position and head in a cache
    if case["kind"] == "read":
        return {"bytes": float(2 * total * kv * (held + dim * size[case["out"]]) + tables), "flops": float(2 * total * kv * dim)}
    if case["kind"] == "append":   # rows in; queries, what the cache then holds and its values out
        values = total * (heads + 2 * kv) * dim
        extra = 4 * ((heads + 2 * kv) * dim * case["bias"] + 2 * dim * case["norm"])
        return {"bytes": float(values * size[case["x"]] + 2 * total * (heads * dim + 2 * kv * dim) + 2 * total * kv * held + extra + tables),
                "flops": float(values * (6 + case["bias"] + 4 * case["norm"]))}
    cached = sum(_distinct(case, n - r, r) for n, r in zip(lens, rows))
    pairs = sum(_pairs(case, n - r, r) for n, r in zip(lens, rows))
    return {"bytes": float(cached * kv * held * 2 + total * heads * dim * (2 + (4 if case["out"] == "f32" else 2)) + tables),
            "flops": 4.0 * dim * heads * pairs}


def _exact_mx(x, fmt):
    """The values that the blocks of float64 rows are held as: the nearest of the codes' values, of two as near the even code's."""
    codes = torch.arange(127 if fmt == "mxf8" else 8, device="cuda")
    bits, bias = (3, 7) if fmt == "mxf8" else (1, 1)
    e, m = codes >> bits, (codes & (1 << bits) - 1).double() / (1 << bits)
    values = torch.where(e > 0, (1 + m) * _two_to(e - bias), m * 2.0 ** (1 - bias))
    block = x.reshape(-1, 32)
    scale = _two_to(((block.abs().amax(1).view(torch.int64) >> 52) - 1023 - (8 if fmt == "mxf8" else 2)).clamp(min=-127))
    y = (block.abs() / scale[:, None]).clamp(max=float(values[-1])).contiguous()
    hi = torch.searchsorted(values, y).clamp(max=len(values) - 1)
    lo = (hi - 1).clamp(min=0)
    below, above = y - values[lo], values[hi] - y
    pick = torch.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)
    return (torch.copysign(values[pick], block) * scale[:, None]).view_as(x)


def _exact_weights(state, first, last):
    """Rows of the matrix in float64, value by value."""
    c = state["w"][first:last].int()
    n = torch.stack([c % 16, c // 16], 2).flatten(1)
    e, m = n % 8 // 2, n % 2
    size = torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * _two_to(e - 1))
    return torch.where(n >= 8, -size, size) * _two_to(state["wp"][first:last].int() - 127).repeat_interleave(32, 1)


@torch.no_grad()
def exact(case, seed):
    """Products a slice of columns at a time, sequences one by one, attention head by head and a block of rows at a time. Quantised
    rows are given as the values that they are held as, but for keys that are appended: after the norm and the rotation the last
    bits of float32 decide where a few of them are rounded to."""
    state = prepare(case, seed)
    f64 = torch.float64
    if case["kind"] == "quantize":
        return {"values": torch.cat([_exact_mx(p.to(f64), case["format"]) for p in state["x"].split(max(1, (1 << 24) // case["cols"]))])}
    if case["kind"] == "linear":
        x = torch.cat([_exact_mx(p.to(f64), case["format"]) for p in state["x"].split(max(1, (1 << 24) // case["inner"]))])
        step = max(1, (1 << 24) // case["inner"])
        y = torch.cat([x @ _exact_weights(state, n, n + step).T.contiguous() for n in range(0, case["cols"], step)], 1)
        return {"y": y if state["bias"] is None else y + state["bias"].to(f64)}
    heads, kv, dim, page = case["heads"], case["kv"], case["dim"], case["page"]
    lens, rows = _shape(case)

    def cached(cache):   # [pages][page size][kv heads][head size]
        n = kv * page * dim
        c = cache[:, :n].reshape(-1, kv, page, dim).int()
        e, m = c % 128 // 8, (c % 8).to(f64) / 8
        y = torch.where(e > 0, (1 + m) * _two_to(e - 7), m * 2.0 ** -6) * torch.where(c > 127, -1, 1)
        return (y * _two_to(cache[:, n:].int() - 127).view(-1, kv, page, dim // 32).repeat_interleave(32, 3)).transpose(1, 2)

    result = {}
    if case["kind"] == "attend":
        k_cache, v_cache = cached(state["k_cache"]), cached(state["v_cache"])
        result["out"] = torch.empty(state["total"], heads, dim, dtype=f64, device="cuda")
    elif case["kind"] == "read":
        caches = {"k": state["k_cache"], "v": state["v_cache"]}
        result = {name: torch.empty(state["total"], kv, dim, dtype=f64, device="cuda") for name in caches}
    else:
        result = {name: torch.empty(state["total"], n, dim, dtype=f64, device="cuda") for name, n in (("q", heads), ("v", kv))}
    row = 0
    for s, (n, new) in enumerate(zip(lens, rows)):
        pos = torch.arange(n - new, n, device="cuda")
        pages = state["table"][s].long()
        if case["kind"] == "append":
            x = state["x"][row:row + new].to(f64)
            if state["bias"] is not None:
                x = x + state["bias"].to(f64)
            parts = list(x.view(new, -1, dim).split([heads, kv, kv], 1))
            freq = torch.exp(-math.log(BASE) * 2 * torch.arange(dim // 2, dtype=f64, device="cuda") / dim)
            turn = torch.polar(torch.ones(new, dim // 2, dtype=f64, device="cuda"), torch.outer(pos.to(f64), freq))[:, None]
            for i, gamma in enumerate((state["q_norm"], state["k_norm"])):
                if gamma is not None:
                    parts[i] = parts[i] / torch.sqrt(parts[i].square().mean(-1, keepdim=True) + EPS) * gamma.to(f64)
                z = torch.complex(parts[i][..., :dim // 2].contiguous(), parts[i][..., dim // 2:].contiguous()) * turn
                parts[i] = torch.cat((z.real, z.imag), -1)
            if state["bias"] is not None:   # (the value that is rounded to eight bits is a float32 sum)
                parts[2] = parts[2].float().to(f64)
            for name, part in (("q", parts[0]), ("v", _exact_mx(parts[2].contiguous(), "mxf8"))):
                result[name][row:row + new] = part
        elif case["kind"] == "read":
            used = pages[:-(-n // page)]
            for name, cache in caches.items():
                result[name][row:row + new] = cached(cache[used]).flatten(0, 1)[:n]
        else:
            keys = torch.arange(n, device="cuda")
            k, v = (c[pages[keys // page], keys % page] for c in (k_cache, v_cache))
            for h in range(heads):
                kh, vh = k[:, h * kv // heads].T.contiguous(), v[:, h * kv // heads].contiguous()
                for b in range(0, new, 2048):
                    p = pos[b:b + 2048, None]
                    hidden = keys > p
                    if case["window"]:
                        hidden |= (keys <= p - case["window"]) & (keys >= case["sinks"])
                    z = state["q"].view(-1, heads, dim)[row + b:row + min(b + 2048, new), h].to(f64) @ kh * dim ** -0.5
                    z[hidden] = -math.inf
                    result["out"][row + b:row + min(b + 2048, new), h] = torch.softmax(z, -1) @ vh
        row += new
    result = {name: y.flatten(1) for name, y in result.items()}
    return {**result, "k": None} if case["kind"] == "append" else result
