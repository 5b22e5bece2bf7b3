"""Timed cases of the key/value cache operators: appending rows with the
position rotation, reading them back, and attention over the cache with a
sliding window and first tokens that stay visible.

A sequence's keys and values live in pages of `page` slots; its page table
row names them in order. A call brings n new rows of a sequence whose length,
those rows included, is L: row j has slot L - n + j. Pages hold bf16, or four
bits a value (e2m1 codes, one power of two for each 32 features).
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEVICE = "cuda"
BASE = 10000.0


def _case(name, op, **kw):
    case = {"name": name, "op": op, "cache": "bf16", "dtype": "bf16", "heads": 20, "kv_heads": 20, "dim": 128,
            "page": 64, "sequences": 1, "rows": 1, "ragged": False, "length": 1, "window": 0, "sinks": 0, "block": 1,
            "rope": 128, "axes": 1, "halves": False}
    case.update(kw)
    return case


def listed():
    return [
        # One new token for each of 16 sequences: the smallest call, all latency.
        _case("append_step_bf16", "append", sequences=16, rows=1, length=200, ragged=True),
        # A prompt of four ragged clips with (t, h, w) positions, 126 of 128
        # features rotated as in the block's layers.
        _case("append_clips_bf16", "append", sequences=4, rows=4096, ragged=True, length=4200, rope=126, axes=3),
        # fp32 activations into four bits, and the rows back as the cache holds them.
        _case("append_read_4bit", "append", cache="4bit", dtype="f32", sequences=2, rows=4096, ragged=True,
              length=4500, heads=32, kv_heads=8, halves=True),
        # One token over a short cache: launches and latency.
        _case("token_short_bf16", "attention", length=700, sequences=1),
        # One token of one very long sequence: work split over the keys.
        _case("token_long_bf16", "attention", length=131072, sequences=1, page=256),
        # A serving batch with shared heads, a window of 4096 and 64 sinks.
        _case("batch_window_bf16", "attention", sequences=64, heads=32, kv_heads=8, length=16384, ragged=True,
              window=4096, sinks=64, page=16),
        # A serving batch over four bits.
        _case("batch_4bit", "attention", cache="4bit", sequences=32, length=16384, ragged=True),
        # Four draft tokens a sequence, shared heads, fp32 activations over four bits.
        _case("drafts_f32_4bit", "attention", cache="4bit", dtype="f32", sequences=16, heads=32, kv_heads=8, rows=4,
              length=8192, ragged=True, window=6000, sinks=4, dim=64),
        # A long clip frame by frame: 16x16 tokens a frame that see each other,
        # four frames back and the 64 text tokens, fp32 activations.
        _case("frames_f32", "attention", dtype="f32", rows=9 * 256, length=64 + 33 * 256, window=1024, sinks=64,
              block=256),
        # A chunk of a prompt behind a window.
        _case("chunk_window_bf16", "attention", sequences=2, rows=4096, length=16384, window=4096, sinks=64,
              ragged=True),
        # A chunk over four bits, shared heads.
        _case("chunk_4bit", "attention", cache="4bit", sequences=3, rows=1500, ragged=True, length=9000, heads=32,
              kv_heads=8),
        # A whole prompt of 16384 tokens: the largest.
        _case("prompt_bf16", "attention", rows=16384, length=16384),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    """Other sizes of the same kinds of work: one token to long prompts, odd
    lengths, shared heads, both cache types, pages of 16 to 256."""
    while True:
        op = rng.choice(["append", "attention", "attention", "attention"])
        heads, kv = rng.choice([(20, 20), (20, 20), (32, 8), (16, 16), (12, 4), (28, 4), (7, 7), (16, 1)])
        dim = rng.choice([128, 128, 128, 64])
        halves, axes = rng.choice([(False, 1), (True, 1), (False, 3)])
        rope = dim if axes == 1 else dim - dim % 6
        case = _case("", op, cache=rng.choice(["bf16", "4bit"]), dtype=rng.choice(["bf16", "bf16", "f32"]),
                     heads=heads, kv_heads=kv, dim=dim, page=rng.choice([16, 32, 64, 128, 256]),
                     ragged=rng.random() < 0.7, rope=rope, axes=axes, halves=halves)
        del case["name"]
        if op == "append":
            case["sequences"] = _log(rng, 1, 100)
            case["rows"] = _log(rng, 1, 12000)
            case["length"] = case["rows"] + rng.randint(0, 300)
            if not 4 <= case["sequences"] * case["rows"] <= 16000:
                continue
            return case
        step = rng.random() < 0.55
        case["sequences"] = _log(rng, 1, 128 if step else 6)
        case["rows"] = rng.choice([1, 1, 1, 2, 3, 5]) if step else _log(rng, 20, 9000)
        case["length"] = case["rows"] + _log(rng, 1, 60000 if step else 16000)
        if rng.random() < 0.5:
            case["window"] = _log(rng, 100, 9000)
            case["sinks"] = rng.choice([0, 1, 4, 58, 64])
            case["block"] = 1 if step else rng.choice([1, 1, 240, 256])
        cached = case["sequences"] * case["length"] * kv * dim
        scores = case["sequences"] * heads * case["rows"] * case["length"]
        if cached > 1.2e9 or scores > 4e9 or case["sequences"] * case["length"] < rng.uniform(0, 1) * 3000:
            continue
        return case


# ---- the inputs ----

def _type(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def _sizes(case):
    """New rows and length of each sequence: fixed by the case, spread from a
    small part of the largest to the largest where it is ragged."""
    n, s = case["rows"], case["sequences"]
    if not case["ragged"]:
        return [n] * s, [case["length"]] * s
    rows = [max(1, n - (n * 3 * i * (i + 1) // (4 * s * (s + 1) or 1)) - (i % 2 if n > 2 else 0)) for i in range(s)]
    before = case["length"] - n
    return rows, [r + before - before * 7 * ((i * 5) % s) // (8 * s) for i, r in enumerate(rows)]


def _encode(x):
    """Four bits a value: codes (two a byte, even feature low) and a byte
    e + 127 for each 32 features, in the input's precision."""
    g = x.reshape(*x.shape[:-1], -1, 32)
    m, e = torch.frexp(g.abs().amax(-1, keepdim=True))
    e = (e - 2 - (m <= 0.875).to(e.dtype)).clamp(min=-126)
    y = torch.ldexp(g, -e)
    a = y.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = (code + 8 * (y < 0)).to(torch.uint8).reshape(x.shape)
    return code[..., 0::2] + 16 * code[..., 1::2], (e.squeeze(-1) + 127).to(torch.uint8)


def _decode(codes, scale):
    """The values that codes stand for, fp32."""
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    mag = (code & 7).float()
    big = torch.ldexp(1.0 + 0.5 * (code & 1), ((code >> 1) & 3).to(torch.int32) - 1)
    value = torch.where(mag < 2, 0.5 * mag, big)
    value = torch.where(code > 7, -value, value)
    s = torch.ldexp(torch.ones((), device=codes.device), scale.to(torch.int32) - 127)
    return (value.reshape(*scale.shape, 32) * s[..., None]).flatten(-2)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    rows, lengths = _sizes(case)
    page, kv, dim, dtype = case["page"], case["kv_heads"], case["dim"], _type(case)
    total, width = sum(rows), -(-max(lengths) // page)
    used = [-(-n // page) for n in lengths]
    pages = sum(used) + 1
    order = torch.randperm(pages, generator=gen, device=DEVICE).to(torch.int32)
    table = torch.full((case["sequences"], width), -1, device=DEVICE, dtype=torch.int32)
    at = 0
    for s, n in enumerate(used):
        table[s, :n] = order[at:at + n]
        at += n

    def normal(*shape, std=1.0, to=dtype):
        return torch.randn(shape, generator=gen, device=DEVICE).mul_(std).to(to)

    state = {"case": case, "total": total, "pages": pages, "width": width, "table": table,
             "lengths": torch.tensor(lengths, device=DEVICE, dtype=torch.int32),
             "cu": torch.tensor([0] + rows, device=DEVICE).cumsum(0).to(torch.int32),
             "rows": max(rows), "longest": max(lengths)}
    # The slots' earlier contents: keys and values of unit scale.
    for name in ("k", "v"):
        parts = [normal(n, kv, page, dim, to=torch.bfloat16) for n in _split(pages, 64 * 1024 * 1024 // (kv * page * dim))]
        if case["cache"] == "bf16":
            state[name + "_pool"] = torch.cat(parts)
        else:
            coded = [_encode(p.float()) for p in parts]
            state[name + "_pool"] = torch.cat([c for c, _ in coded])
            state[name + "_scale"] = torch.cat([s for _, s in coded])
    state["q"] = normal(total, case["heads"], dim, std=2.0)
    state["out"] = torch.empty_like(state["q"])
    if case["op"] == "append":
        state["k"], state["v"] = normal(total, kv, dim), normal(total, kv, dim)
        # Positions as a long session has them: far from zero, apart from the slots.
        far = torch.randint(0, 1 << (20 if case["axes"] == 1 else 7), (total, case["axes"]), generator=gen,
                            device=DEVICE)
        state["positions"] = far.to(torch.int32)
        if case["cache"] != "bf16":
            for name in ("k_rows", "v_rows"):
                state[name] = torch.empty(total, kv, dim, device=DEVICE, dtype=torch.bfloat16)
    return state


def _split(n, most):
    most = max(1, most)
    return [min(most, n - i) for i in range(0, n, most)]


# ---- the framework's calls ----

def _handles(state):
    """Descriptors, the rotation and the workspace, made once as a program does."""
    sys.path.insert(0, os.path.abspath("seedvr2-ncnn_amd"))
    import awa_hip as A

    A.init(0)
    case = state["case"]
    size = 4 if case["dtype"] == "f32" else 2
    four = case["cache"] != "bf16"

    def blob(name, heads, elemsize):
        return A.mat(state[name].data_ptr(), case["dim"], heads, state["total"], elemsize, dims=3)

    cache = A.KvCache(A.KV_MXFP4 if four else A.KV_BF16, state["pages"], case["page"], case["kv_heads"], case["dim"],
                      state["k_pool"].data_ptr(), state["v_pool"].data_ptr(), state["table"].data_ptr(),
                      case["sequences"], state["width"], state["lengths"].data_ptr(),
                      k_scale=state["k_scale"].data_ptr() if four else 0,
                      v_scale=state["v_scale"].data_ptr() if four else 0)
    rows = A.KvRows(state["rows"], state["cu"].data_ptr())
    h = {"A": A, "cache": cache, "rows": rows, "q": blob("q", case["heads"], size),
         "out": blob("out", case["heads"], size)}
    if case["op"] == "append":
        h["k"], h["v"] = blob("k", case["kv_heads"], size), blob("v", case["kv_heads"], size)
        h["rope"] = A.Rope(case["rope"], case["axes"], BASE, halves=case["halves"])
        if four:
            h["k_rows"], h["v_rows"] = blob("k_rows", case["kv_heads"], 2), blob("v_rows", case["kv_heads"], 2)
    else:
        h["mask"] = A.KvMask(case["window"], case["sinks"], case["block"], state["longest"])
        h["scale"] = case["dim"] ** -0.5
        nbytes = A.kv_attention_workspace(cache, rows, h["q"], h["mask"])
        h["workspace"] = torch.empty(max(nbytes, 16), device=DEVICE, dtype=torch.uint8)
        h["nbytes"] = nbytes
    return h


def _run_own(state):
    if "handles" not in state:
        state["handles"] = _handles(state)
    h = state["handles"]
    A = h["A"]
    if state["case"]["op"] == "attention":
        A.kv_attention(h["cache"], h["rows"], h["q"], h["mask"], h["scale"], h["out"], h["workspace"].data_ptr(),
                       h["nbytes"])
        return {"out": state["out"]}
    A.kv_append(h["cache"], h["rows"], h["k"], h["v"], h["rope"], state["positions"].data_ptr(), q=h["q"],
                q_out=h["out"])
    if state["case"]["cache"] == "bf16":
        return {"q": state["out"], "k": state["k_pool"], "v": state["v_pool"]}
    A.kv_read(h["cache"], h["rows"], h["k_rows"], h["v_rows"])
    return {"q": state["out"], "k": state["k_rows"], "v": state["v_rows"]}


# ---- the plain form ----

def _rotate(x, positions, case):
    """Angles and rotation in 64 bits: far positions, and values next to a
    border of the four-bit codes."""
    rope, axes = case["rope"], case["axes"]
    pairs = rope // axes // 2
    freq = BASE ** (-torch.arange(pairs, device=x.device, dtype=torch.float64) / pairs)
    angle = (positions.double()[:, :, None] * freq).flatten(1)[:, None]
    cos, sin = angle.cos(), angle.sin()
    x = x.double()
    a, b = (x[..., :rope // 2], x[..., rope // 2:rope]) if case["halves"] else (x[..., 0:rope:2], x[..., 1:rope:2])
    u, w = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat([u, w], -1) if case["halves"] else torch.stack([u, w], -1).flatten(-2)
    return torch.cat([turned, x[..., rope:]], -1)


def _places(state):
    """Sequence, slot and index in it of each new row."""
    cu, lengths = state["cu"].long(), state["lengths"].long()
    t = torch.arange(state["total"], device=DEVICE)
    s = torch.searchsorted(cu, t, right=True) - 1
    j = t - cu[s]
    return s, lengths[s] - (cu[s + 1] - cu[s]) + j, j


def _run_append(state):
    case = state["case"]
    q = _rotate(state["q"], state["positions"], case)
    k = _rotate(state["k"], state["positions"], case)
    state["out"].copy_(q)
    s, slot, _ = _places(state)
    page, at = state["table"][s, slot // case["page"]].long(), slot % case["page"]
    if case["cache"] == "bf16":
        state["k_pool"][page, :, at] = k.to(torch.bfloat16)
        state["v_pool"][page, :, at] = state["v"].to(torch.bfloat16)
        return {"q": state["out"], "k": state["k_pool"], "v": state["v_pool"]}
    for name, x in (("k", k), ("v", state["v"].float())):
        codes, scale = _encode(x)
        state[name + "_pool"][page, :, at] = codes
        state[name + "_scale"][page, :, at] = scale
        state[name + "_rows"].copy_(_decode(state[name + "_pool"][page, :, at], state[name + "_scale"][page, :, at]))
    return {"q": state["out"], "k": state["k_rows"], "v": state["v_rows"]}


def _cached(state, name):
    """[sequences, kv heads, slots, dim] in fp32; slots behind a length are 0."""
    case = state["case"]
    table = state["table"].long().clamp(min=0)
    x = state[name + "_pool"][table]
    x = x.float() if case["cache"] == "bf16" else _decode(x, state[name + "_scale"][table])
    x = x.transpose(1, 2).flatten(2, 3)
    there = torch.arange(x.shape[2], device=DEVICE) < state["lengths"][:, None]
    return torch.where(there[:, None, :, None], x, x.new_zeros(()))


def _run_attention(state):
    case = state["case"]
    s, slot, j = _places(state)
    kv, group, dim = case["kv_heads"], case["heads"] // case["kv_heads"], case["dim"]
    q = torch.zeros(case["sequences"], state["rows"], kv, group, dim, device=DEVICE)
    q[s, j] = state["q"].float().reshape(-1, kv, group, dim)
    q = q.permute(0, 2, 1, 3, 4).flatten(2, 3)
    keys = _cached(state, "k")
    scores = torch.matmul(q, keys.transpose(2, 3).contiguous()).mul_(dim ** -0.5)
    del keys
    first = state["lengths"] - (state["cu"][1:] - state["cu"][:-1])
    p = first[:, None] + torch.arange(state["rows"], device=DEVICE)
    end = case["sinks"] - torch.div(case["sinks"] - 1 - p, case["block"], rounding_mode="floor") * case["block"]
    begin = end - case["window"] if case["window"] else torch.zeros_like(end)
    key = torch.arange(scores.shape[-1], device=DEVICE)
    seen = (key < end[..., None]) & (key < state["lengths"][:, None, None])
    seen &= (key >= begin[..., None]) | (key < case["sinks"])
    seen = seen[:, None].repeat_interleave(group, 2)
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = scores.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights, _cached(state, "v")) / torch.where(total == 0, torch.ones_like(total), total)
    out = out.reshape(case["sequences"], kv, state["rows"], group, dim).transpose(1, 2).flatten(2, 3)
    state["out"].copy_(out[s, j])
    return {"out": state["out"]}


def run(state):
    if own:
        return _run_own(state)
    return _run_append(state) if state["case"]["op"] == "append" else _run_attention(state)


# ---- what a pass cannot do without ----

def _span(p, length, case):
    """Visible keys of the row at slot p: (sinks seen, begin, end)."""
    end = case["sinks"] + case["block"] * -(-(p + 1 - case["sinks"]) // case["block"])
    begin = max(0, end - case["window"]) if case["window"] else 0
    end = min(end, length)
    return min(case["sinks"], begin, end), min(begin, end), end


def work(case):
    rows, lengths = _sizes(case)
    size = 4 if case["dtype"] == "f32" else 2
    kv, heads, dim = case["kv_heads"], case["heads"], case["dim"]
    cached = 2 * kv * (2 * dim if case["cache"] == "bf16" else dim // 2 + dim // 32)
    total = sum(rows)
    if case["op"] == "append":
        moved = total * (size * dim * (2 * heads + 2 * kv) + cached + 4 * case["axes"])
        if case["cache"] != "bf16":
            moved += total * (cached + 2 * kv * dim * 2)
        return {"bytes": moved, "flops": total * (heads + kv) * case["rope"] * 3}
    seen = pairs = 0
    for n, length in zip(rows, lengths):
        last = _span(length - 1, length, case)
        first = _span(length - n, length, case)
        seen += last[2] - min(first[1], last[2]) + min(last[0], first[1])
        step = case["block"] if case["block"] > 1 else max(1, n // 64)
        at = list(range(length - n, length, step))
        for p in at:
            a, b, e = _span(p, length, case)
            pairs += (a + e - b) * min(step, length - p)
    return {"bytes": seen * cached + 2 * total * heads * dim * size, "flops": 4.0 * dim * heads * pairs}


# ---- the same in 64 bits, from the definitions ----

def _turned(x, positions, case):
    """x e^(i angle), each pair of features as one complex number."""
    x, rope = x.double(), case["rope"]
    per_axis = rope // case["axes"]
    out = x.clone()
    for axis in range(case["axes"]):
        for i in range(per_axis // 2):
            angle = positions[:, axis].double() * math.pow(BASE, -2.0 * i / per_axis)
            lo = i if case["halves"] else axis * per_axis + 2 * i
            hi = lo + rope // 2 if case["halves"] else lo + 1
            z = torch.complex(x[..., lo], x[..., hi]) * torch.polar(torch.ones_like(angle), angle)[:, None]
            out[..., lo], out[..., hi] = z.real, z.imag
    return out


def _nearest(x):
    """x as the nearest of the four-bit values, ties to the even code."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=x.device, dtype=torch.float64)
    middle = (grid[1:] + grid[:-1]) / 2
    middle[1::2] = torch.nextafter(middle[1::2], torch.zeros_like(middle[1::2]))
    g = x.double().unflatten(-1, (-1, 32))
    top = g.abs().amax(-1, keepdim=True)
    e = torch.full_like(top, -126.0)
    for k in range(-126, 127):
        e = torch.where(top > 7.0 * 2.0 ** k, torch.full_like(e, k + 1.0), e)
    unit = torch.pow(2.0, e)
    return (torch.sign(g) * grid[torch.bucketize((g / unit).abs(), middle)] * unit).flatten(-2)


def exact(case, seed):
    state = prepare(case, seed)
    rows, lengths = _sizes(case)
    page, dim = case["page"], case["dim"]
    if case["op"] == "append":
        q, k, v = _turned(state["q"], state["positions"], case), _turned(state["k"], state["positions"], case), None
        v = state["v"].double()
        if case["cache"] != "bf16":
            return {"q": q, "k": _nearest(k), "v": _nearest(v)}
        pools = {name: state[name + "_pool"].double() for name in ("k", "v")}
        at = 0
        for s, (n, length) in enumerate(zip(rows, lengths)):
            slots = torch.arange(length - n, length, device=DEVICE)
            where = state["table"][s].long()[slots // page], slots % page
            for name, x in (("k", k), ("v", v)):
                pools[name][where[0], :, where[1]] = x[at:at + n]
            at += n
        return {"q": q, **pools}
    out = torch.zeros(state["total"], case["heads"], dim, device=DEVICE, dtype=torch.float64)
    group, at = case["heads"] // case["kv_heads"], 0
    for s, (n, length) in enumerate(zip(rows, lengths)):
        where = state["table"][s, :-(-length // page)].long()
        key = torch.arange(length, device=DEVICE)
        spans = torch.tensor([_span(p, length, case) for p in range(length - n, length)], device=DEVICE)
        seen = (key < spans[:, :1]) | ((key >= spans[:, 1:2]) & (key < spans[:, 2:]))
        for h in range(case["kv_heads"]):
            kv = []
            for name in ("k", "v"):
                x = state[name + "_pool"][where, h]
                if case["cache"] != "bf16":
                    values = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6],
                                          device=DEVICE, dtype=torch.float64)
                    x = values[torch.stack([x % 16, x // 16], -1).long()].flatten(-2).unflatten(-1, (-1, 32))
                    x = (x * torch.pow(2.0, state[name + "_scale"][where, h].double() - 127)[..., None]).flatten(-2)
                kv.append(x.double().flatten(0, 1)[:length])
            for i in range(h * group, (h + 1) * group):
                s_ = (state["q"][at:at + n, i].double() @ kv[0].t()) * dim ** -0.5
                s_ = s_.masked_fill_(~seen, -math.inf)
                s_ = s_.sub_(s_.amax(-1, keepdim=True)).exp_()
                out[at:at + n, i] = (s_ @ kv[1]) / s_.sum(-1, keepdim=True)
        at += n
    return {"out": out}
