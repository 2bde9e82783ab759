"""Cases that measure the paged-cache operators (`instantllm_amd.paged.PagedAttention`).

Keys and values live in pages of a shared cache; a table per sequence names its pages. Two calls
belong to each layer of a model that serves several requests at once:

  append   the new rows' queries, keys and values: bias, a norm for each head, the rotation by
           position; keys and values go to their places in the cache, queries to a buffer
  attend   the new rows' attention over their sequences' cached positions (their own included),
           either all earlier ones or a sliding window and the first few (`sinks`)

A sequence's new rows are its last ones: row i of n stands at position len - n + i. Head layouts
are (query heads, key/value heads, head size): (14, 2, 64) is the model that the engine serves.
"""
import functools
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LAYOUTS = [(14, 2, 64), (32, 8, 128), (12, 12, 64), (16, 1, 128), (28, 4, 128)]
BASE, EPS = 1e6, 1e-6


def listed():
    return [
        # one decode step of the engine's model: the product before it gives float32, with a bias to add
        {"name": "append_step", "kind": "append", "heads": 14, "kv": 2, "dim": 64, "type": "f16", "x": "f32", "page": 16,
         "seqs": 1, "rows": 1, "lo": 257, "hi": 257, "bias": True, "norm": False, "mix": 1},
        # a decode step of 64 requests, with head norms
        {"name": "append_batch64", "kind": "append", "heads": 32, "kv": 8, "dim": 128, "type": "bf16", "x": "bf16", "page": 32,
         "seqs": 64, "rows": 1, "lo": 2, "hi": 700, "bias": False, "norm": True, "mix": 2},
        # the engine's longest prompt chunk
        {"name": "append_chunk4096", "kind": "append", "heads": 14, "kv": 2, "dim": 64, "type": "f16", "x": "f16", "page": 64,
         "seqs": 1, "rows": 4096, "lo": 8200, "hi": 8200, "bias": True, "norm": False, "mix": 3},
        # ragged prompts of a batch
        {"name": "append_ragged7", "kind": "append", "heads": 32, "kv": 8, "dim": 128, "type": "bf16", "x": "bf16", "page": 16,
         "seqs": 7, "rows": 5000, "lo": 3500, "hi": 6100, "bias": False, "norm": True, "mix": 4},
        # decode steps: one short request (float32 out, as the product after it takes it), one very long one
        {"name": "step_1x500", "kind": "attend", "heads": 14, "kv": 2, "dim": 64, "type": "f16", "out": "f32", "page": 16,
         "seqs": 1, "rows": 1, "lo": 500, "hi": 500, "window": 0, "sinks": 0, "mix": 5},
        {"name": "step_1x131071", "kind": "attend", "heads": 14, "kv": 2, "dim": 64, "type": "f16", "out": "f16", "page": 64,
         "seqs": 1, "rows": 1, "lo": 131071, "hi": 131071, "window": 0, "sinks": 0, "mix": 6},
        # decode steps of batches: contexts of very different lengths, and long ones through a window
        {"name": "step_64_ragged", "kind": "attend", "heads": 32, "kv": 8, "dim": 128, "type": "bf16", "out": "bf16", "page": 16,
         "seqs": 64, "rows": 1, "lo": 100, "hi": 9000, "window": 0, "sinks": 0, "mix": 7},
        {"name": "step_200_window", "kind": "attend", "heads": 14, "kv": 2, "dim": 64, "type": "f16", "out": "f16", "page": 32,
         "seqs": 200, "rows": 1, "lo": 300, "hi": 20000, "window": 1024, "sinks": 4, "mix": 8},
        # prompts: a short one, a chunk of a long one through a window, a mixed batch (prompts' chunks
        # beside single tokens), a long one
        {"name": "prompt_333", "kind": "attend", "heads": 14, "kv": 2, "dim": 64, "type": "f16", "out": "f16", "page": 16,
         "seqs": 1, "rows": 333, "lo": 333, "hi": 333, "window": 0, "sinks": 0, "mix": 9},
        {"name": "prompt_4096_window", "kind": "attend", "heads": 14, "kv": 2, "dim": 64, "type": "f16", "out": "f16", "page": 64,
         "seqs": 1, "rows": 4096, "lo": 8200, "hi": 8200, "window": 1024, "sinks": 4, "mix": 10},
        {"name": "prompt_mixed9", "kind": "attend", "heads": 32, "kv": 8, "dim": 128, "type": "bf16", "out": "bf16", "page": 16,
         "seqs": 9, "rows": 700, "lo": 400, "hi": 5000, "window": 0, "sinks": 0, "mix": 11},
        {"name": "prompt_8000", "kind": "attend", "heads": 28, "kv": 4, "dim": 128, "type": "bf16", "out": "bf16", "page": 128,
         "seqs": 1, "rows": 8000, "lo": 8000, "hi": 8000, "window": 0, "sinks": 0, "mix": 12},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    heads, kv, dim = rng.choice(LAYOUTS)
    case = {"heads": heads, "kv": kv, "dim": dim, "type": rng.choice(["f16", "bf16"]), "page": rng.choice([16, 32, 64, 128, 256]),
            "mix": rng.randrange(1 << 20)}
    what = rng.choice(["append", "append", "step", "step", "prompt", "prompt"])
    if what == "append":
        seqs = _log_int(rng, 1, 64)
        rows = rng.choice([1, _log_int(rng, 2, 12000 // seqs)])
        lo = rows + rng.randint(0, 300)
        return {**case, "kind": "append", "x": rng.choice(["f32", case["type"]]), "seqs": seqs, "rows": rows, "lo": lo,
                "hi": lo + _log_int(rng, 1, 500), "bias": rng.random() < 0.5, "norm": rng.random() < 0.5}
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
    new row, the others any number up to `rows`. They belong to the case, not to the inputs' seed."""
    rng = random.Random(case["mix"])
    lens = [case["hi"]] + [_log_int(rng, case["lo"], case["hi"]) for _ in range(case["seqs"] - 1)]
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
    return PagedAttention(heads, kv, dim, page_size=page, dtype=dtype, rope_base=BASE, norm_eps=EPS)


def prepare(case, seed):
    heads, kv, dim, dt = case["heads"], case["kv"], case["dim"], DTYPES[case["type"]]
    lens, rows = _shape(case)
    table, pages = _tables(case, seed)
    gen = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    total = sum(rows)
    state = {"case": case, "k_cache": normal(pages, case["page"], kv, dim).to(dt), "v_cache": normal(pages, case["page"], kv, dim).to(dt),
             "lens": torch.tensor(lens, dtype=torch.int32).cuda(), "table": table.cuda(), "pages": pages,
             "row0": torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], dtype=torch.int32).cuda(), "total": total, "most": max(rows),
             "handle": _handle(heads, kv, dim, case["page"], case["type"]) if own else None}
    if case["kind"] == "append":
        state.update(x=normal(total, (heads + 2 * kv) * dim).to(DTYPES[case["x"]]), q=torch.empty(total, heads * dim, dtype=dt, device="cuda"),
                     bias=normal((heads + 2 * kv) * dim) if case["bias"] else None,
                     q_norm=1 + 0.2 * normal(dim) if case["norm"] else None, k_norm=1 + 0.2 * normal(dim) if case["norm"] else None)
    else:   # some queries' scores are nearly even, others' fall on a few keys
        state.update(q=(normal(total, heads, dim) * (0.5 + 3 * torch.rand(total, heads, 1, generator=gen, device="cuda"))).to(dt).view(total, -1),
                     out=torch.empty(total, heads * dim, dtype=DTYPES[case["out"]], device="cuda"))
    return state


# ---- the plain forms -----------------------------------------------------------------------
def _places(state):
    """Each new row's sequence and position."""
    counts = state["row0"][1:] - state["row0"][:-1]
    seq = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), counts.long(), output_size=state["total"])
    at = torch.arange(state["total"], device="cuda") - state["row0"][seq]
    return seq, at, state["lens"][seq] - counts[seq] + at


def _plain_append(state):
    case = state["case"]
    heads, kv, dim, page = case["heads"], case["kv"], case["dim"], case["page"]
    seq, _, pos = _places(state)
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

    where = state["table"][seq, torch.div(pos, page, rounding_mode="floor")].long() * page + pos % page
    state["k_cache"].view(-1, kv, dim)[where] = turn(k).to(state["k_cache"].dtype)
    state["v_cache"].view(-1, kv, dim)[where] = v.to(state["v_cache"].dtype)
    state["q"].copy_(turn(q).view(-1, heads * dim))
    return {"q": state["q"], "k_cache": state["k_cache"], "v_cache": state["v_cache"]}


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
    k = state["k_cache"][pick].reshape(seqs, longest, kv, dim).transpose(1, 2).float()
    v = state["v_cache"][pick].reshape(seqs, longest, kv, dim).transpose(1, 2).float()
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
def _own_append(state):
    case = state["case"]
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    x, size, width = state["x"], state["x"].element_size(), (heads + 2 * kv) * dim
    h = state["handle"]
    address = x.data_ptr()
    h.append(_batch(state), state["k_cache"].data_ptr(), state["v_cache"].data_ptr(), q=address, k=address + heads * dim * size,
             v=address + (heads + kv) * dim * size, q_out=state["q"].data_ptr(), x_dtype=case["x"], x_stride=width,
             bias=state["bias"].data_ptr() if case["bias"] else None, q_norm=state["q_norm"].data_ptr() if case["norm"] else None,
             k_norm=state["k_norm"].data_ptr() if case["norm"] else None)
    return {"q": state["q"], "k_cache": state["k_cache"], "v_cache": state["v_cache"]}


def _own_attend(state):
    case = state["case"]
    state["handle"].attend(_batch(state), state["k_cache"].data_ptr(), state["v_cache"].data_ptr(), state["q"].data_ptr(),
                           state["out"].data_ptr(), out_dtype=case["out"], window=case["window"], sinks=case["sinks"])
    return {"out": state["out"]}


def _batch(state):
    """The batch as the calls take it: device addresses and sizes."""
    return state["handle"].batch(lens=state["lens"].data_ptr(), table=state["table"].data_ptr(), table_width=state["table"].shape[1],
                                 pages=state["pages"], seqs=state["case"]["seqs"], rows=state["total"], row0=state["row0"].data_ptr(),
                                 max_rows=state["most"])


@torch.no_grad()
def run(state):
    if state["case"]["kind"] == "append":
        return _own_append(state) if own else _plain_append(state)
    return _own_attend(state) if own else _plain_attend(state)


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
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    lens, rows = _shape(case)
    total = sum(rows)
    tables = 4 * (2 * case["seqs"] + 1 + sum(-(-n // case["page"]) for n in lens))
    if case["kind"] == "append":
        values = total * (heads + 2 * kv) * dim
        wide = 4 if case["x"] == "f32" else 2
        extra = 4 * ((heads + 2 * kv) * dim * case["bias"] + 2 * dim * case["norm"])
        return {"bytes": float(values * (wide + 2) + extra + tables), "flops": float(values * (3 + case["bias"] + 4 * case["norm"]))}
    cached = sum(_distinct(case, n - r, r) for n, r in zip(lens, rows))
    pairs = sum(_pairs(case, n - r, r) for n, r in zip(lens, rows))
    return {"bytes": float(cached * kv * dim * 2 * 2 + total * heads * dim * (2 + (4 if case["out"] == "f32" else 2)) + tables),
            "flops": 4.0 * dim * heads * pairs}


@torch.no_grad()
def exact(case, seed):
    """Sequence by sequence in float64; attention head by head, a block of rows at a time."""
    state = prepare(case, seed)
    heads, kv, dim, page = case["heads"], case["kv"], case["dim"], case["page"]
    lens, rows = _shape(case)
    f64 = torch.float64
    cached = [state["k_cache"].to(f64), state["v_cache"].to(f64)]
    result = torch.empty(state["total"], heads, dim, dtype=f64, device="cuda")
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
            result[row:row + new] = parts[0]
            for c, part in zip(cached, parts[1:]):
                c[pages[pos // page], pos % page] = part
        else:
            keys = torch.arange(n, device="cuda")
            k, v = (c[pages[keys // page], keys % page] for c in cached)
            for h in range(heads):
                kh, vh = k[:, h * kv // heads].T.contiguous(), v[:, h * kv // heads].contiguous()
                for b in range(0, new, 2048):
                    p = pos[b:b + 2048, None]
                    hidden = keys > p
                    if case["window"]:
                        hidden |= (keys <= p - case["window"]) & (keys >= case["sinks"])
                    z = state["q"].view(-1, heads, dim)[row + b:row + min(b + 2048, new), h].to(f64) @ kh * dim ** -0.5
                    z[hidden] = -math.inf
                    result[row + b:row + min(b + 2048, new), h] = torch.softmax(z, -1) @ vh
        row += new
    result = result.view(state["total"], -1)
    return {"q": result, "k_cache": cached[0], "v_cache": cached[1]} if case["kind"] == "append" else {"out": result}
