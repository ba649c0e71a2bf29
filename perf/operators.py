"""The serving operators of a paged 8-bit key/value cache, as measured work.

Four operators, in the order a serving step calls them:

* ``plan``    block tables, positions and slot maps from the requests' lengths
* ``rope``    rotary positions on the query and key heads
* ``append``  rotary positions and the write of the step's keys and values into
  the cache: e4m3 values, one power-of-two scale per page and head
* ``attend``  causal attention of every request's new tokens over its pages

With ``own`` false ``run`` computes them in elementary torch operations; with
``own`` true it calls the framework's ``paged`` module.  Both take the same
tensors.
"""
import math
import os
import sys

import torch

own = False

PKG = "hot-cold-neural-split-openinfer2_b200"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
E_MIN, E_MAX = -40, 40              # exponents a page scale can take
_paged = None


def _framework():
    global _paged
    if _paged is None:
        path = os.path.abspath(PKG)
        if path not in sys.path:
            sys.path.insert(0, path)
        import paged
        _paged = paged
    return _paged


# ─── Cases ────────────────────────────────────────────────────────────────────
def listed():
    gqa = {"nq": 32, "nkv": 8, "dim": 128}
    return [
        # one decode step of a full batch: a token each, tables of 8192 positions
        {"name": "plan decode 64", "op": "plan", "requests": 64, "q_lo": 1, "q_hi": 1, "start_lo": 17,
         "start_hi": 8000, "page": 64, "width": 128, "pad": 0},
        # a step that admits many prompts of all lengths, small pages, rows padded as for a captured step
        {"name": "plan prompts 256", "op": "plan", "requests": 256, "q_lo": 1, "q_hi": 256, "start_lo": 0,
         "start_hi": 3900, "page": 16, "width": 260, "pad": 1000},
        # the smallest call: one token of one request
        {"name": "rope 1 token", "op": "rope", "tokens": 1, "rotary": 128, "interleaved": False, "dtype": "f16",
         "far": 8192, **gqa},
        # a prompt's layer
        {"name": "rope 8192 tokens", "op": "rope", "tokens": 8192, "rotary": 128, "interleaved": False,
         "dtype": "bf16", "far": 8192, **gqa},
        # half of the head rotated, neighbouring pairs, positions of a long context
        {"name": "rope part 2047 tokens", "op": "rope", "tokens": 2047, "rotary": 64, "interleaved": True,
         "dtype": "f16", "far": 131072, **gqa},
        # a decode step's write: 64 requests, most of them inside a page
        {"name": "append decode 64", "op": "append", "requests": 64, "q_lo": 1, "q_hi": 1, "start_lo": 0,
         "start_hi": 300, "page": 64, "rotary": 128, "interleaved": False, "dtype": "f16", **gqa},
        # prompts' write: ragged, small pages
        {"name": "append prompts 6", "op": "append", "requests": 6, "q_lo": 100, "q_hi": 2048, "start_lo": 0,
         "start_hi": 500, "page": 16, "rotary": 128, "interleaved": False, "dtype": "bf16", **gqa},
        # the latency case: one token of one request
        {"name": "attend 1 token", "op": "attend", "requests": 1, "q_lo": 1, "q_hi": 1, "start_lo": 512,
         "start_hi": 512, "page": 64, "dtype": "f16", **gqa},
        # a decode batch with ragged contexts
        {"name": "attend decode 64", "op": "attend", "requests": 64, "q_lo": 1, "q_hi": 1, "start_lo": 100,
         "start_hi": 8000, "page": 64, "dtype": "bf16", **gqa},
        # few requests with long contexts
        {"name": "attend long 4", "op": "attend", "requests": 4, "q_lo": 1, "q_hi": 1, "start_lo": 60000,
         "start_hi": 131070, "page": 64, "dtype": "f16", **gqa},
        # a prompt in one piece
        {"name": "attend prompt 4096", "op": "attend", "requests": 1, "q_lo": 4096, "q_hi": 4096, "start_lo": 0,
         "start_hi": 0, "page": 64, "dtype": "f16", **gqa},
        # prompts in pieces behind what is cached: small heads, eight query heads to a key head
        {"name": "attend pieces 5", "op": "attend", "requests": 5, "q_lo": 33, "q_hi": 1500, "start_lo": 0,
         "start_hi": 8000, "page": 128, "dtype": "bf16", "nq": 16, "nkv": 2, "dim": 64},
    ]


def draw(rng):
    def log_int(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))

    op = rng.choice(["plan", "rope", "append", "attend", "attend"])
    nkv = rng.choice([1, 2, 4, 8])
    heads = {"nq": nkv * rng.choice([1, 2, 4, 7, 8]), "nkv": nkv, "dim": rng.choice([64, 128])}
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["f16", "bf16"])
    if op == "plan":
        q_hi = log_int(1, 256)
        start = log_int(1, 3900)
        return {"op": op, "requests": log_int(1, 256), "q_lo": 1, "q_hi": q_hi, "start_lo": rng.randint(0, start),
                "start_hi": start, "page": page, "width": (start + q_hi) // page + 1 + rng.randint(0, 40),
                "pad": rng.randint(0, 300)}
    rotary = rng.choice([heads["dim"], heads["dim"] // 2, 2 * rng.randint(1, heads["dim"] // 2)])
    if op == "rope":
        return {"op": op, "tokens": log_int(1, 8192), "rotary": rotary, "interleaved": rng.random() < 0.5,
                "dtype": dtype, "far": log_int(16, 131072), **heads}
    if op == "append":
        q_hi = log_int(1, 2048)
        return {"op": op, "requests": log_int(1, 64 if q_hi < 100 else 6), "q_lo": rng.randint(1, q_hi),
                "q_hi": q_hi, "start_lo": 0, "start_hi": rng.randint(0, 500), "page": page, "rotary": rotary,
                "interleaved": rng.random() < 0.5, "dtype": dtype, **heads}
    if rng.random() < 0.5:                       # decode: one or a few tokens a request
        far = log_int(16, 100000)
        q_hi = rng.choice([1, 1, 1, 2, 5])
        return {"op": op, "requests": log_int(1, max(1, min(64, 250000 // far))), "q_lo": 1, "q_hi": q_hi,
                "start_lo": rng.randint(0, far), "start_hi": far, "page": page, "dtype": dtype, **heads}
    q_hi = log_int(2, 1500)
    return {"op": op, "requests": rng.randint(1, 4), "q_lo": rng.randint(1, q_hi), "q_hi": q_hi, "start_lo": 0,
            "start_hi": log_int(1, 4000), "page": page, "dtype": dtype, **heads}


def _lengths(case):
    """(cached, new) tokens of every request: spread over the case's ranges, the ends included."""
    n = case["requests"]

    def spread(lo, hi, step):
        if n == 1:
            return [hi]
        at = [(i * step) % 1.0 for i in range(n)]
        top, low = max(at), min(at)
        return [lo + int((hi - lo) * (a - low) / (top - low) + 0.5) for a in at]

    return (spread(case["start_lo"], case["start_hi"], 0.6180339887498949),
            spread(case["q_lo"], case["q_hi"], 0.7548776662466927))


def work(case):
    if case["op"] == "plan":
        starts, new = _lengths(case)
        p = case["page"]
        touched = sum((s + q + p - 1) // p - s // p for s, q in zip(starts, new))
        rows = sum(new) + case["pad"]
        return {"bytes": 8 * len(new) + 4 * touched + 8 * len(new) + 4 + 16 * rows, "flops": 4 * rows}
    heads = case["nq"] + 2 * case["nkv"]
    if case["op"] == "rope":
        t, n = case["tokens"], case["nq"] + case["nkv"]
        return {"bytes": t * (n * case["dim"] * 4 + case["rotary"] * 4 + 8), "flops": t * n * case["rotary"] * 3}
    starts, new = _lengths(case)
    t = sum(new)
    if case["op"] == "append":
        d, kv = case["dim"], 2 * case["nkv"]
        p = case["page"]
        pages = sum((s + q + p - 1) // p - s // p for s, q in zip(starts, new))
        return {"bytes": t * (heads * d * 2 + case["nq"] * d * 2 + kv * d + case["rotary"] * 4 + 16) + pages * kv * 8,
                "flops": t * ((case["nq"] + case["nkv"]) * case["rotary"] * 3 + kv * d * 2)}
    keys = sum(s + q for s, q in zip(starts, new))
    pairs = sum(q * s + q * (q + 1) // 2 for s, q in zip(starts, new))
    pages = sum((s + q + case["page"] - 1) // case["page"] for s, q in zip(starts, new))
    return {"bytes": keys * case["nkv"] * 2 * case["dim"] + pages * (4 + 8 * case["nkv"])
            + t * case["nq"] * case["dim"] * 4, "flops": 4 * case["dim"] * case["nq"] * pairs}


# ─── Inputs ───────────────────────────────────────────────────────────────────
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(1000003 + int(seed))


def _quantise(x):
    """e4m3 values and the power-of-two scale of each [..., tokens, dim] block of x (fp32)."""
    top = x.abs().amax(dim=(-2, -1))
    mantissa, exponent = torch.frexp(top)
    exponent = torch.where(mantissa > 0.875, exponent - 8, exponent - 9).clamp(E_MIN, E_MAX)
    exponent = torch.where(top == 0, torch.full_like(exponent, E_MIN), exponent)
    scale = torch.ldexp(torch.ones_like(top), exponent)
    return (x / scale[..., None, None]).to(torch.float8_e4m3fn), scale


def _tables(starts, new, page, width, spare, g):
    """Block tables over a shuffled pool of pages: every request's cached part is in place."""
    held = [(s + page - 1) // page for s in starts]
    want = [(s + q + page - 1) // page for s, q in zip(starts, new)]
    n_pages = sum(want) + spare
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    column = torch.arange(width, device="cuda")[None]
    count = torch.tensor(held, device="cuda")[:, None]
    base = torch.tensor([sum(held[:i]) for i in range(len(held))], device="cuda")[:, None]
    at = (base + column).clamp(max=n_pages - 1)
    tables = torch.where(column < count, order[at], torch.full_like(order[at], -1))
    return tables, order, sum(held), n_pages


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _rotary_tables(rows, rotary):
    frequency = 500000.0 ** (-torch.arange(rotary // 2, device="cuda", dtype=torch.float64) / (rotary // 2))
    angle = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * frequency
    return angle.cos().float(), angle.sin().float()


def _full_tables(starts, new, page, g):
    """Tables with every page of the step in place, positions, slots and the row offsets."""
    width = max((s + q + page - 1) // page for s, q in zip(starts, new))
    n_pages = sum((s + q + page - 1) // page for s, q in zip(starts, new))
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    tables = torch.full((len(new), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    positions, slots, cu = [], [], [0]
    for r, (s, q) in enumerate(zip(starts, new)):
        n = (s + q + page - 1) // page
        tables[r, :n] = order[at:at + n]
        at += n
        pos = torch.arange(s, s + q, device="cuda")
        positions.append(pos)
        slots.append(tables[r][pos // page].long() * page + pos % page)
        cu.append(cu[-1] + q)
    return tables, torch.cat(positions), torch.cat(slots), _ints(cu), n_pages


def prepare(case, seed):
    g = _generator(seed)
    if case["op"] == "plan":
        starts, new = _lengths(case)
        tables, order, held, n_pages = _tables(starts, new, case["page"], case["width"], 64, g)
        free = torch.full((n_pages,), -1, dtype=torch.int32, device="cuda")
        free[:n_pages - held] = order[held:].flip(0)
        return {"op": "plan", "starts": _ints(starts), "new": _ints(new), "tables": tables, "free": free,
                "n_free": _ints([n_pages - held]), "page": case["page"], "rows": sum(new) + case["pad"]}
    dt = DTYPES[case["dtype"]]
    nq, nkv, d = case["nq"], case["nkv"], case["dim"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["op"] == "rope":
        t = case["tokens"]
        cos, sin = _rotary_tables(case["far"], case["rotary"])
        positions = torch.randint(0, case["far"], (t,), generator=g, device="cuda")
        # rows of one fused projection: heads are views of it, as in the engine
        qkv = normal(t, nq + 2 * nkv, d).to(dt)
        return {"op": "rope", "q": qkv[:, :nq], "k": qkv[:, nq:nq + nkv], "cos": cos, "sin": sin,
                "positions": positions, "interleaved": case["interleaved"]}
    starts, new = _lengths(case)
    page = case["page"]
    tables, positions, slots, cu_q, n_pages = _full_tables(starts, new, page, g)
    k_pages, k_scale = _quantise(normal(n_pages, nkv, page, d))
    v_pages, v_scale = _quantise(normal(n_pages, nkv, page, d) * 0.7 + 0.05)
    state = {"op": case["op"], "k_pages": k_pages.view(torch.uint8), "v_pages": v_pages.view(torch.uint8),
             "k_scale": k_scale, "v_scale": v_scale}
    t = sum(new)
    if case["op"] == "append":
        cos, sin = _rotary_tables(max(s + q for s, q in zip(starts, new)), case["rotary"])
        qkv = normal(t, nq + 2 * nkv, d)
        qkv[:, nq:nq + nkv] *= 1 + normal(t, 1, 1).abs()       # some tokens above what their page holds
        qkv = qkv.to(dt)
        return {**state, "q": qkv[:, :nq], "k": qkv[:, nq:nq + nkv], "v": qkv[:, nq + nkv:], "cos": cos, "sin": sin,
                "positions": positions, "slots": slots, "interleaved": case["interleaved"]}
    return {**state, "q": normal(t, nq, d).to(dt), "tables": tables, "cu_q": cu_q, "max_q": max(new),
            "kv_lens": _ints([s + q for s, q in zip(starts, new)])}


# ─── The operators in plain form ──────────────────────────────────────────────
def _plain_plan(s):
    starts, new, tables, page = s["starts"].long(), s["new"].long(), s["tables"], s["page"]
    kv = starts + new
    column = torch.arange(tables.shape[1], device="cuda")[None]
    inside = (column >= (starts // page)[:, None]) & (column < ((kv + page - 1) // page)[:, None])
    missing = inside & (tables < 0)
    rank = missing.flatten().cumsum(0).view(missing.shape)
    taken = s["free"][(s["n_free"].long() - rank).clamp(min=0)]
    tables.copy_(torch.where(missing, taken, tables))
    s["n_free"].sub_(missing.sum().int())
    cu = torch.cat([new.new_zeros(1), new.cumsum(0)])
    t = torch.arange(s["rows"], device="cuda")
    r = torch.searchsorted(cu[1:].contiguous(), t, right=True).clamp(max=len(new) - 1)
    pos = starts[r] + t - cu[r]
    behind = t >= cu[-1]
    pos = torch.where(behind, torch.full_like(pos, -1), pos)
    at = pos.clamp(min=0)
    slots = torch.where(behind, pos, tables[r, at // page].long() * page + at % page)
    return {"cu_q": cu.int(), "kv_lens": kv.int(), "positions": pos, "slots": slots, "tables": tables,
            "n_free": s["n_free"]}


def _plain_rotate(x, c, s, interleaved, dtype):
    """x [T, heads, dim] rotated by the angles of c, s [T, rotary / 2], rounded once."""
    half = c.shape[1]
    x = x.to(dtype)
    c, s = c[:, None].to(dtype), s[:, None].to(dtype)
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack((a * c - b * s, a * s + b * c), dim=-1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat((a * c - b * s, a * s + b * c), dim=-1)
    return torch.cat((turned, x[..., 2 * half:]), dim=-1)


def _plain_write(pages, scales, x, slots):
    """The rows x [T, heads, dim] (16 bits) into their slots of the pages, in place."""
    n_pages, heads, page, dim = pages.shape
    held = slots // page
    x = x.float()
    top = x.abs().amax(-1)                                                  # [T, heads]
    first = torch.full((n_pages,), page, device="cuda").scatter_reduce(0, held, slots % page, "amin")
    most = top.new_zeros(n_pages, heads).index_reduce(0, held, top, "amax")
    mantissa, exponent = torch.frexp(most)
    exponent = torch.where(mantissa > 0.875, exponent - 8, exponent - 9).clamp(E_MIN, E_MAX)
    exponent = torch.where(most == 0, torch.full_like(exponent, E_MIN), exponent)
    need = torch.ldexp(torch.ones_like(most), exponent)
    new = torch.where((first == 0)[:, None], need, torch.maximum(need, scales))
    new = torch.where((first == page)[:, None], scales, new)                # pages that no token enters
    values = pages.view(torch.float8_e4m3fn).float()
    before = torch.arange(page, device="cuda")[None] < torch.where(first == page, torch.zeros_like(first), first)[:, None]
    again = (values * (scales / new)[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    pages.copy_(torch.where(before[:, None, :, None], again, pages))
    scales.copy_(new)
    pages[held, :, slots % page] = (x / new[held][..., None]).to(torch.float8_e4m3fn).view(torch.uint8)


def _plain_attend(s):
    q, cu, kv, tables = s["q"], s["cu_q"].long(), s["kv_lens"].long(), s["tables"]
    _, nkv, page, dim = s["k_pages"].shape
    t, nq, _ = q.shape
    group, n = nq // nkv, tables.shape[0]
    at = tables.clamp(min=0).long()

    def dense(pages, scales):
        x = pages.view(torch.float8_e4m3fn)[at].float() * scales[at][..., None, None]     # [n, pages, nkv, page, dim]
        return x.transpose(1, 2).reshape(n, nkv, -1, dim)

    keys, values = dense(s["k_pages"], s["k_scale"]), dense(s["v_pages"], s["v_scale"])
    token = torch.arange(t, device="cuda")
    r = torch.searchsorted(cu[1:].contiguous(), token, right=True)
    row = token - cu[r]
    new = cu[1:] - cu[:-1]
    padded = torch.zeros(n, s["max_q"], nq, dim, device="cuda")
    padded[r, row] = q.float()
    padded = padded.view(n, -1, nkv, group, dim).permute(0, 2, 3, 1, 4)                    # [n, nkv, group, rows, dim]
    score = torch.matmul(padded, keys[:, :, None].transpose(-1, -2)) * (1.0 / math.sqrt(dim))
    last = (kv - new)[:, None] + torch.arange(s["max_q"], device="cuda")[None]             # [n, rows]
    seen = torch.arange(keys.shape[2], device="cuda") <= last[..., None]                   # [n, rows, keys]
    seen = seen & (torch.arange(keys.shape[2], device="cuda") < kv[:, None, None])
    score = score.masked_fill(~seen[:, None, None], float("-inf"))
    weight = (score - score.amax(-1, keepdim=True)).exp()
    weight = weight / weight.sum(-1, keepdim=True)
    out = torch.matmul(weight, values[:, :, None])                                         # [n, nkv, group, rows, dim]
    out = out.permute(0, 3, 1, 2, 4).reshape(n, -1, nq, dim)
    return out[r, row].to(q.dtype)


def run(s):
    if s["op"] == "plan":
        if own:
            cu_q, kv_lens, positions, slots = _framework().page_plan(s["starts"], s["new"], s["tables"], s["free"],
                                                                     s["n_free"], s["page"], s["rows"])
            return {"cu_q": cu_q, "kv_lens": kv_lens, "positions": positions, "slots": slots, "tables": s["tables"],
                    "n_free": s["n_free"]}
        return _plain_plan(s)
    if s["op"] == "rope":
        if own:
            q, k = _framework().rope(s["q"], s["k"], s["cos"], s["sin"], s["positions"], interleaved=s["interleaved"])
            return {"q": q, "k": k}
        c, sn = s["cos"][s["positions"]], s["sin"][s["positions"]]
        return {"q": _plain_rotate(s["q"], c, sn, s["interleaved"], torch.float32).to(s["q"].dtype),
                "k": _plain_rotate(s["k"], c, sn, s["interleaved"], torch.float32).to(s["k"].dtype)}
    if s["op"] == "append":
        if own:
            q = _framework().rope_append(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["positions"], s["slots"],
                                         s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"],
                                         interleaved=s["interleaved"])
        else:
            c, sn = s["cos"][s["positions"]], s["sin"][s["positions"]]
            q = _plain_rotate(s["q"], c, sn, s["interleaved"], torch.float32).to(s["q"].dtype)
            # the key's rounding decides its byte: values next to a border, in 64 bits
            k = _plain_rotate(s["k"], c, sn, s["interleaved"], torch.float64).to(s["k"].dtype)
            _plain_write(s["k_pages"], s["k_scale"], k, s["slots"])
            _plain_write(s["v_pages"], s["v_scale"], s["v"], s["slots"])
        return {"q": q, "k_pages": s["k_pages"].view(torch.float8_e4m3fn), "k_scale": s["k_scale"],
                "v_pages": s["v_pages"].view(torch.float8_e4m3fn), "v_scale": s["v_scale"]}
    if own:
        return {"out": _framework().paged_attention(s["q"], s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"],
                                                    s["tables"], s["cu_q"], s["kv_lens"], max_q=s["max_q"])}
    return {"out": _plain_attend(s)}


# ─── The definitions in 64 bits ───────────────────────────────────────────────
def _exact_turn(x, c, s, interleaved):
    """The rotation as a product of complex numbers."""
    n = 2 * c.shape[1]
    part = x[..., :n].double()
    pair = part.unflatten(-1, (-1, 2)) if interleaved else part.unflatten(-1, (2, -1)).transpose(-1, -2)
    turned = torch.view_as_complex(pair.contiguous()) * torch.complex(c.double(), s.double())[:, None]
    turned = torch.view_as_real(turned)
    out = x.double().clone()
    out[..., :n] = turned.flatten(-2) if interleaved else turned.transpose(-1, -2).flatten(-2)
    return out


def _exact_write(pages, scales, x, slots):
    """Page by page: the scale that the page needs, then its rows."""
    page = pages.shape[2]
    pages, scales = pages.view(torch.float8_e4m3fn).float().double(), scales.double()
    rungs = torch.arange(E_MIN, E_MAX + 1, device="cuda")
    ladder = torch.ldexp(torch.ones(len(rungs), dtype=torch.float64, device="cuda"), rungs)
    order = slots // page
    for p in torch.unique(order).tolist():
        rows = (order == p).nonzero()[:, 0]
        at = slots[rows] % page
        top = x[rows].abs().amax(dim=(0, 2))
        # the first power of two that holds it, by comparison: a logarithm may fall on the wrong side of a whole number
        need = ladder[torch.searchsorted(448 * ladder, top)]
        lo = int(at.min())
        new = need if lo == 0 else torch.maximum(need, scales[p])
        if lo:
            kept = pages[p, :, :lo] * (scales[p] / new)[:, None, None]
            pages[p, :, :lo] = kept.float().to(torch.float8_e4m3fn).float().double()
        scales[p] = new
        # a 16-bit value over a power of two is exact in 32 bits
        pages[p][:, at] = (x[rows] / new[None, :, None]).float().to(torch.float8_e4m3fn).float().double().transpose(0, 1)
    return pages, scales


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "plan":
        return None
    if case["op"] == "rope":
        c, sn = s["cos"][s["positions"]], s["sin"][s["positions"]]
        return {"q": _exact_turn(s["q"], c, sn, s["interleaved"]), "k": _exact_turn(s["k"], c, sn, s["interleaved"])}
    if case["op"] == "append":
        c, sn = s["cos"][s["positions"]], s["sin"][s["positions"]]
        q = _exact_turn(s["q"], c, sn, s["interleaved"])
        k = _exact_turn(s["k"], c, sn, s["interleaved"]).to(s["k"].dtype).double()
        kp, ks = _exact_write(s["k_pages"], s["k_scale"], k, s["slots"])
        vp, vs = _exact_write(s["v_pages"], s["v_scale"], s["v"].double(), s["slots"])
        return {"q": q, "k_pages": kp, "k_scale": ks, "v_pages": vp, "v_scale": vs}
    q, cu, kv = s["q"], s["cu_q"].tolist(), s["kv_lens"].tolist()
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    page = case["page"]
    group = case["nq"] // case["nkv"]
    k_all, v_all = (s[n].view(torch.float8_e4m3fn) for n in ("k_pages", "v_pages"))
    for r in range(len(kv)):
        lo, hi, n = cu[r], cu[r + 1], kv[r]
        mine = s["tables"][r, :(n + page - 1) // page].long()
        after = torch.arange(n, device="cuda")[None] > torch.arange(n - (hi - lo), n, device="cuda")[:, None]
        for h in range(case["nkv"]):
            k = (k_all[mine, h].double() * s["k_scale"][mine, h].double()[:, None, None]).flatten(0, 1)[:n]
            v = (v_all[mine, h].double() * s["v_scale"][mine, h].double()[:, None, None]).flatten(0, 1)[:n]
            for j in range(h * group, (h + 1) * group):
                score = q[lo:hi, j].double() @ k.T / math.sqrt(case["dim"])
                out[lo:hi, j] = torch.softmax(score.masked_fill(after, -math.inf), dim=-1) @ v
    return {"out": out}
