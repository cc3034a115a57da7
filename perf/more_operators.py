"""Performance cases of what a serving step does around the paged key-value
cache: the plan of pages and slots, norms and position rotation of the new
tokens on their way into the pages, and a cache of 4-bit microscaled rows
(append, read, attention of single tokens and of prompts).

Each case is one pass through one operator (``op``) at the sizes it gives.  With
``own`` false a pass computes it with elementary torch operations in 32 bits
(angles in 64); with ``own`` true it calls the package.  Lengths of the sequences
of a case are spread between ``ragged`` times the case's length and the whole of
it, in an order that the seed draws.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # magnitudes of 4-bit codes: sign, two bits of exponent, one of fraction


def listed():
    return [
        # Two conversations near their start, few narrow heads: launch and latency.
        {"name": "token_small", "op": "token", "batch": 2, "heads": 8, "kv": 2, "dim": 64, "rows": 301, "ragged": 0.7,
         "type": "bf16", "page": 16, "sinks": 0, "window": -1, "weights": False},
        # A served batch at mid length.
        {"name": "token_batch", "op": "token", "batch": 64, "heads": 32, "kv": 8, "dim": 128, "rows": 8200,
         "ragged": 0.3, "type": "bf16", "page": 32, "sinks": 0, "window": -1, "weights": False},
        # A few long documents whose rows' weights are gathered for a later eviction.
        {"name": "token_long", "op": "token", "batch": 3, "heads": 32, "kv": 4, "dim": 128, "rows": 131071,
         "ragged": 0.5, "type": "f16", "page": 64, "sinks": 0, "window": -1, "weights": True},
        # Whole prompts, causal.
        {"name": "prompt_causal", "op": "prompt", "batch": 2, "heads": 16, "kv": 4, "dim": 128, "new": 4096,
         "before": 0, "ragged": 1.0, "type": "bf16", "page": 64, "sinks": 0, "window": -1},
        # Next turns of several conversations, with a sliding window and first rows that stay visible.
        {"name": "prompt_turns", "op": "prompt", "batch": 5, "heads": 24, "kv": 8, "dim": 96, "new": 301,
         "before": 5000, "ragged": 0.1, "type": "f16", "page": 16, "sinks": 4, "window": 1500},
        # One new row for each sequence of a batch of young conversations; the rows are read back.
        {"name": "store_token", "op": "store", "batch": 128, "kv": 8, "dim": 128, "new": 1, "before": 20,
         "ragged": 1.0, "type": "bf16", "page": 32},
        # Prompts of a batch; the rows are read back.
        {"name": "store_prompt", "op": "store", "batch": 4, "kv": 8, "dim": 128, "new": 4096, "before": 0,
         "ragged": 0.5, "type": "bf16", "page": 64},
        # The keys of a long document, for the graph over them.
        {"name": "read_keys", "op": "read", "rows": 60001, "kv": 8, "dim": 128, "page": 64, "f32": True,
         "values": False},
        # One token of each served sequence.
        {"name": "rotate_token", "op": "rotate", "tokens": 48, "heads": 32, "kv": 8, "dim": 128, "rotary": 128,
         "pairs": "halves", "norm": True, "type": "bf16", "page": 32, "far": 8000},
        # A chunk of prompts, far into long documents, part of the dims rotated.
        {"name": "rotate_prompt", "op": "rotate", "tokens": 12001, "heads": 32, "kv": 8, "dim": 128, "rotary": 64,
         "pairs": "halves", "norm": True, "type": "bf16", "page": 64, "far": 900000},
        # A step of single tokens: few sequences begin a page.
        {"name": "plan_token", "op": "plan", "batch": 200, "new": 1, "before": 4000, "ragged": 0.1, "ends": 0.0,
         "page": 16, "spare": 1.0},
        # A step that ends some sequences and takes in prompts, more than there are pages for.
        {"name": "plan_prompt", "op": "plan", "batch": 96, "new": 6000, "before": 300, "ragged": 0.05, "ends": 0.1,
         "page": 16, "spare": 0.8},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng: random.Random):
    op = rng.choice(["token", "token", "token", "prompt", "prompt", "store", "read", "rotate", "rotate", "plan"])
    kv = rng.choice([1, 2, 4, 8])
    c = {"op": op, "page": rng.choice([16, 32, 64, 128]), "ragged": rng.choice([0.1, 0.5, 1.0])}
    if op in ("token", "prompt", "store", "read"):
        c["kv"], c["dim"] = kv, rng.choice([64, 64, 96, 128, 128, 128, 160, 256])
    if op in ("token", "prompt", "store", "rotate"):
        c["type"] = rng.choice(["bf16", "f16"])
    sinks, window = rng.choice([(0, -1), (0, -1), (rng.randint(0, 8), rng.randint(100, 2000))])
    if op == "token":
        c["heads"] = kv * rng.choice([1, 2, 4, 7, 8, 16])
        c["rows"] = _log(rng, 30, 131072)
        c["batch"] = _log(rng, 1, min(64, max(1.0, 4e8 / (2 * c["rows"] * kv * c["dim"]))))
        c["weights"] = rng.random() < 0.4
        c["sinks"], c["window"] = sinks, window
    elif op == "prompt":
        c["heads"] = kv * rng.choice([1, 2, 4, 8])
        c["new"] = _log(rng, 2, 8000)
        c["before"] = rng.choice([0, _log(rng, 10, 20000)])
        most = 16 * 4096 * 4096 * 2 * 128 / (c["heads"] * c["dim"])
        if c["new"] * (c["before"] + c["new"]) > most:
            c["new"], c["before"] = min(c["new"], 1000), min(c["before"], 2000)
        c["batch"] = _log(rng, 1, min(8, max(1.0, most / (c["new"] * (c["before"] + c["new"])))))
        c["sinks"], c["window"] = sinks, window
    elif op == "store":
        c["new"] = rng.choice([1, _log(rng, 2, 4096)])
        c["before"] = rng.randint(0, 500)
        c["batch"] = _log(rng, 1, min(64, max(1.0, 1.6e7 / ((c["new"] + c["before"]) * kv * c["dim"]))))
    elif op == "read":
        c["rows"] = _log(rng, 3, min(100000, 6e7 / (kv * c["dim"])))
        c["f32"], c["values"] = rng.random() < 0.5, rng.random() < 0.5
        del c["ragged"]
    elif op == "rotate":
        c["kv"], c["dim"] = kv, rng.choice([64, 80, 96, 128, 128, 256])
        c["heads"] = kv * rng.choice([1, 2, 4, 7, 8])
        c["tokens"] = _log(rng, 1, min(20000, 6e7 / (c["dim"] * (c["heads"] + 2 * kv))))
        c["rotary"] = rng.choice([0, 16, 32, 64, c["dim"], c["dim"], c["dim"]])
        c["pairs"] = rng.choice(["halves", "halves", "neighbours"])
        c["norm"] = rng.random() < 0.7
        c["far"] = _log(rng, 100, 1000000)
        del c["ragged"]
    else:
        c["batch"] = _log(rng, 1, 512)
        c["new"] = rng.choice([1, 1, _log(rng, 2, 500000 // c["batch"])])
        c["before"] = _log(rng, 1, 20000)
        c["ends"] = rng.choice([0.0, 0.2])
        c["spare"] = rng.choice([0.5, 1.0])
    return c


def _spread(most, ragged, batch):
    """Lengths from ragged * most to most, evenly spread."""
    least = max(1, int(most * ragged))
    return [most - (most - least) * b // max(1, batch - 1) for b in range(batch)]


def _new_and_all(case):
    """New rows and all rows of each sequence of a case."""
    if case["op"] == "token":
        rows = _spread(case["rows"], case["ragged"], case["batch"])
        return [1] * len(rows), rows
    new = _spread(case["new"], case["ragged"], case["batch"])
    return new, [n + case["before"] for n in new]


# ---- inputs --------------------------------------------------------------------
def _quantized(x):
    """4-bit rows of x [..., dim]: bytes of two codes each (the even dim's below), a byte's power of two for 32 dims."""
    x = x.float()
    g = x.view(*x.shape[:-1], -1, 32)
    top = g.abs().amax(-1).contiguous().view(torch.int32)
    # the largest value's exponent, one more from a significand of 1.75 on, which would round above 6
    scale = (((top + (1 << 21)) >> 23) - 2).clamp(2, 252)
    y = torch.ldexp(g, (127 - scale).unsqueeze(-1)).view(x.shape)
    m = y.abs()
    code = torch.zeros_like(m, dtype=torch.uint8)
    # halves between neighbours; a tie goes to the even code
    for i, (half, even_below) in enumerate(((0.25, True), (0.75, False), (1.25, True), (1.75, False), (2.5, True),
                                            (3.5, False), (5.0, True))):
        code += (m > half) if even_below else (m >= half)
    code |= (y < 0).to(torch.uint8) << 3
    return code[..., 0::2] | code[..., 1::2] << 4, scale.to(torch.uint8)


def _values(codes, scales):
    """f32 values [..., dim] of 4-bit rows."""
    grid = torch.tensor(GRID + tuple(-v for v in GRID), device=DEV)
    v = torch.stack([grid[(codes & 15).int()], grid[(codes >> 4).int()]], -1).view(*codes.shape[:-1], -1)
    s = torch.ldexp(torch.ones((), device=DEV), scales.int() - 127)
    return (v.view(*scales.shape, 32) * s.unsqueeze(-1)).view(v.shape)


def _pool(s, g, pages, kv, page, dim):
    """A cache of normal rows in 4 bits."""
    for name in ("keys", "values"):
        x = torch.randn((pages, kv, page, dim), generator=g, device=DEV, dtype=torch.bfloat16)
        s[name], s[name[:-1] + "_scales"] = _quantized(x)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    s = {"case": dict(case)}
    return {"plan": _prepare_plan, "rotate": _prepare_rotate, "read": _prepare_read}.get(case["op"], _prepare_cache)(case, s, g)


def _prepare_cache(case, s, g):
    batch, kv, dim, page, op = case["batch"], case["kv"], case["dim"], case["page"], case["op"]
    dt = DTYPES[case["type"]]
    order = torch.randperm(batch, generator=g, device=DEV)
    new, rows = (torch.tensor(v, dtype=torch.int32, device=DEV)[order].contiguous() for v in _new_and_all(case))
    most = max(_new_and_all(case)[1])
    per = -(-most // page)
    ids = torch.randperm(batch * per + 3, generator=g, device=DEV).to(torch.int32)
    s.update(lengths=rows, max_length=most, table=ids[: batch * per].view(batch, per), new=new,
             max_new=max(_new_and_all(case)[0]), tokens=sum(_new_and_all(case)[0]))
    _pool(s, g, batch * per + 3, kv, page, dim)
    if op != "token":
        s["offsets"] = torch.nn.functional.pad(new.cumsum(0), (1, 0)).to(torch.int32)
        s["token"] = torch.arange(s["tokens"], device=DEV)
    if op == "store":
        s["starts"] = rows - new
        s["k"], s["v"] = (torch.randn((s["tokens"], kv, dim), generator=g, device=DEV, dtype=dt) for _ in range(2))
        s["all"] = torch.arange((batch * per + 3) * page, device=DEV)
    else:
        s["q"] = torch.randn((s["tokens"], case["heads"], dim), generator=g, device=DEV, dtype=dt) * 2
        s["window"] = None if case["window"] < 0 else case["window"]
        s["weights"] = torch.rand((batch, kv, per * page), generator=g, device=DEV) if case.get("weights") else None
    return s


def _prepare_read(case, s, g):
    pages = -(-case["rows"] // case["page"])
    _pool(s, g, pages + 3, case["kv"], case["page"], case["dim"])
    page = torch.randperm(pages + 3, generator=g, device=DEV)
    row = torch.arange(case["rows"], device=DEV)
    s["slots"] = page[row // case["page"]] * case["page"] + row % case["page"]
    s["dtype"] = torch.float32 if case["f32"] else torch.bfloat16
    return s


def _prepare_rotate(case, s, g):
    n, heads, kv, dim, page = case["tokens"], case["heads"], case["kv"], case["dim"], case["page"]
    dt = DTYPES[case["type"]]
    # three sequences: ends of long documents; the last tokens are padding of no sequence
    padding = n // 50
    i = torch.arange(n, device=DEV)
    part = i * 3 // max(1, n)
    far = torch.randint(case["far"] // 2, case["far"], (3,), generator=g, device=DEV)
    s["positions"] = torch.where(i < n - padding, far[part] + i, -1).to(torch.int32)
    pages = -(-n // page) + 2
    slot = torch.randperm(pages, generator=g, device=DEV)[i // page] * page + i % page
    s["slots"] = torch.where(i < n - padding, slot, -1)
    s["q"], s["k"], s["v"] = (torch.randn((n, h, dim), generator=g, device=DEV, dtype=dt) * 3 for h in (heads, kv, kv))
    s["keys"], s["values"] = (torch.randn((pages, kv, page, dim), generator=g, device=DEV, dtype=dt) for _ in range(2))
    weights = [1 + 0.2 * torch.randn(dim, generator=g, device=DEV) for _ in range(2)]
    s["q_weight"], s["k_weight"] = (w.to(dt) for w in weights) if case["norm"] else (None, None)
    r = case["rotary"]
    s["frequencies"] = 10000.0 ** (-torch.arange(0, r, 2, device=DEV, dtype=torch.float64) / r) if r else None
    return s


def _prepare_plan(case, s, g):
    batch, page = case["batch"], case["page"]
    order = torch.randperm(batch, generator=g, device=DEV)
    new = torch.tensor(_spread(case["new"], case["ragged"], batch), dtype=torch.int32, device=DEV)[order]
    length = torch.tensor(_spread(case["before"], case["ragged"], batch), dtype=torch.int32, device=DEV)
    length = length[torch.randperm(batch, generator=g, device=DEV)]
    ends = torch.arange(batch, device=DEV) < int(case["ends"] * batch)
    s["new"] = torch.where(ends[torch.randperm(batch, generator=g, device=DEV)], -1, new)
    columns = -(-(case["before"] + case["new"]) // page)
    # an eviction left every seventh sequence one page more than its rows need
    extra = (torch.arange(batch, device=DEV) % 7 == 0).int()
    s["lengths"] = length.contiguous()
    s["held"] = torch.minimum(-(-length // page) + extra, torch.tensor(columns, device=DEV)).int()
    used = -(-case["before"] // page) + 1
    spare = int(case["spare"] * batch * -(-case["new"] // page))
    s["pages"] = batch * used + spare
    ids = torch.randperm(s["pages"], generator=g, device=DEV).to(torch.int32)
    table = torch.full((batch, columns), -1, dtype=torch.int32, device=DEV)
    width = min(used, columns)
    table[:, :width] = ids[: batch * used].view(batch, used)[:, :width]
    s["table"] = torch.where(torch.arange(columns, device=DEV) < s["held"][:, None], table, -1)
    s["free"] = torch.cat([ids[batch * used:], torch.full((batch * used,), -1, dtype=torch.int32, device=DEV)])
    s["count"] = torch.full((1,), spare, dtype=torch.int32, device=DEV)
    s["tokens"] = sum(_spread(case["new"], case["ragged"], batch))
    return s


# ---- plain forms ---------------------------------------------------------------
def _gather(s, what, rows):
    """Rows [batch, n] of the cache as f32 [batch, kv, n, dim]."""
    page = s["case"]["page"]
    p = torch.gather(s["table"], 1, rows // page).long()
    return _values(s[what][p, :, rows % page], s[what[:-1] + "_scales"][p, :, rows % page]).transpose(1, 2)


def _softmax(x, seen):
    """(p, 1 / sum p or 0, log of the sum of exp) over the last axis, of the places that `seen` marks."""
    x = torch.where(seen, x, -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(x - m)
    total = p.sum(-1, keepdim=True)
    return p, torch.where(total > 0, 1.0 / total, 0.0), (m + torch.log(total)).squeeze(-1)


def _token(s):
    c, lens = s["case"], s["lengths"].long()[:, None]
    batch, kv, dim, heads = c["batch"], c["kv"], c["dim"], c["heads"]
    j = torch.arange(s["max_length"], device=DEV)
    seen = j < lens
    if s["window"] is not None:
        seen = seen & ((j < c["sinks"]) | (j >= lens - s["window"]))
    rows = torch.where(seen, j, 0)
    q = s["q"].float().view(batch, kv, heads // kv, dim)
    x = torch.matmul(q, _gather(s, "keys", rows).transpose(-1, -2)) / math.sqrt(dim)
    p, inv, lse = _softmax(x, seen[:, None, None])
    out = (torch.matmul(p, _gather(s, "values", rows)) * inv).view(batch, heads, dim).to(s["q"].dtype)
    got = [out, lse.view(batch, heads)]
    if s["weights"] is not None:
        s["weights"][..., : s["max_length"]] += (p * inv).sum(2)
        got.append(s["weights"])
    return got


def _prompt(s):
    c, lens = s["case"], s["lengths"].long()
    batch, kv, dim, heads, n = c["batch"], c["kv"], c["dim"], c["heads"], s["max_new"]
    off, new = s["offsets"].long(), s["new"].long()[:, None]
    i = torch.arange(n, device=DEV).expand(batch, -1)
    token = torch.where(i < new, off[:-1, None] + i, 0)
    q = s["q"].float()[token].view(batch, n, kv, heads // kv, dim).permute(0, 2, 3, 1, 4)
    pos = (lens[:, None] - new + i)[:, :, None]
    j = torch.arange(s["max_length"], device=DEV)
    seen = (j <= pos) & (j < lens[:, None, None])
    if s["window"] is not None:
        seen &= (j < c["sinks"]) | (j > pos - s["window"])
    rows = torch.where(j < lens[:, None], j, 0)
    k, v = _gather(s, "keys", rows).unsqueeze(2), _gather(s, "values", rows).unsqueeze(2)
    p, inv, lse = _softmax(torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(dim), seen[:, None, None])
    out = (torch.matmul(p, v) * inv).permute(0, 3, 1, 2, 4).reshape(batch * n, heads, dim)
    at = torch.repeat_interleave(torch.arange(batch, device=DEV), s["new"].long(), output_size=s["tokens"])
    real = at * n + s["token"] - off[at]
    return [out[real].to(s["q"].dtype), lse.permute(0, 3, 1, 2).reshape(batch * n, heads)[real]]


def _store(s):
    c = s["case"]
    b = torch.repeat_interleave(torch.arange(c["batch"], device=DEV), s["new"].long(), output_size=s["tokens"])
    row = s["starts"].long()[b] + s["token"] - s["offsets"].long()[b]
    at, slot = s["table"][b, row // c["page"]].long(), row % c["page"]
    s["keys"][at, :, slot], s["key_scales"][at, :, slot] = _quantized(s["k"])
    s["values"][at, :, slot], s["value_scales"][at, :, slot] = _quantized(s["v"])
    return [_values(s[x], s[x[:-1] + "_scales"]).transpose(1, 2).reshape(-1, c["kv"], c["dim"]).to(torch.bfloat16)
            for x in ("keys", "values")]


def _read(s):
    page = s["case"]["page"]
    p, slot = s["slots"] // page, s["slots"] % page
    return [_values(s[x][p, :, slot], s[x[:-1] + "_scales"][p, :, slot]).to(s["dtype"])
            for x in (("keys", "values") if s["case"]["values"] else ("keys",))]


def _turned(s, x, weight):
    c = s["case"]
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * weight.float()
    r = c["rotary"]
    if r:
        angle = s["positions"].double()[:, None] * s["frequencies"]
        cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
        z = y[..., :r]
        a, b = (z[..., : r // 2], z[..., r // 2:]) if c["pairs"] == "halves" else (z[..., 0::2], z[..., 1::2])
        z = [a * cos - b * sin, a * sin + b * cos]
        z = torch.cat(z, -1) if c["pairs"] == "halves" else torch.stack(z, -1).flatten(-2)
        y = torch.cat([z, y[..., r:]], -1)
    return y.to(x.dtype)


def _rotate(s):
    real = s["positions"] >= 0
    q = torch.where(real[:, None, None], _turned(s, s["q"], s["q_weight"]), 0.0)
    k, page = _turned(s, s["k"], s["k_weight"]), s["case"]["page"]
    # places of no token are written with what lies in the first one's
    at = torch.where(s["slots"] >= 0, s["slots"], s["slots"][0])
    token = torch.where(s["slots"] >= 0, torch.arange(real.numel(), device=DEV), 0)
    s["keys"][at // page, :, at % page] = k[token]
    s["values"][at // page, :, at % page] = s["v"][token]
    return [q, s["keys"], s["values"]]


def _before(x):
    return x.cumsum(0) - x


def _plan(s):
    page, tokens, batch = s["case"]["page"], s["tokens"], s["case"]["batch"]
    columns = s["table"].shape[1]
    length, held, asked = s["lengths"].long(), s["held"].long(), s["new"].long()
    new = asked.clamp(min=0)
    first = _before(new)
    fits = (length + new <= columns * page) & (first + new <= tokens)
    grow = torch.where(fits, new, 0)
    after = torch.where(asked < 0, 0, length + grow)
    target = -(-after // page)
    gives, needs = (held - target).clamp(min=0), (target - held).clamp(min=0)
    available = s["count"].long() + gives.sum()
    served = (needs == 0) | (needs.cumsum(0) <= available)
    granted = torch.where(served, grow, 0)
    after = torch.where(asked < 0, 0, length + granted)
    column = torch.arange(columns, device=DEV)
    # pages that are given back, in order, then those that are taken from the top
    out = (column >= target[:, None]) & (column < held[:, None])
    free = torch.cat([s["free"], s["free"][:1]])
    place = s["count"].long() + _before(gives)[:, None] + column - target[:, None]
    free[torch.where(out, place, free.numel() - 1)] = s["table"]
    into = (column >= held[:, None]) & (column < target[:, None]) & served[:, None]
    place = available - 1 - (_before(needs)[:, None] + column - held[:, None])
    s["free"].copy_(free[:-1])
    s["table"].copy_(torch.where(into, free[place.clamp(min=0)], s["table"]))
    taken = torch.where(served, needs, 0)
    b = torch.arange(tokens, device=DEV)
    b = torch.searchsorted(new.cumsum(0), b, right=True).clamp(max=batch - 1)
    i = torch.arange(tokens, device=DEV) - first[b]
    within = (i >= 0) & (i < new[b])
    there = within & (i < granted[b])
    row = torch.where(there, length[b] + i, 0)
    slot = s["table"][b, row // page].long() * page + row % page
    offsets = torch.cat([first, new.sum()[None]])
    held = torch.where(served, target, held)
    ints = (after, held, available - taken.sum(), granted, offsets, torch.where(there, row, -1), torch.where(within, b, -1))
    return [*(x.to(torch.int32) for x in ints), torch.where(there, slot, -1), s["table"], s["free"]]


def run(s):
    op, c = s["case"]["op"], s["case"]
    if not own:
        return {"token": _token, "prompt": _prompt, "store": _store, "read": _read, "rotate": _rotate, "plan": _plan}[op](s)
    from shear_amd import kvcache as KV

    if op == "plan":
        p = KV.plan(c["page"], s["table"], s["lengths"], s["held"], s["new"], s["free"], s["count"], s["tokens"])
        return [p.lengths, p.held, p.count, p.granted, p.offsets, p.positions, p.sequences, p.slots, s["table"], s["free"]]
    if "cache" not in s:
        if op == "rotate":
            s["cache"] = KV.KvCache(s["keys"], s["values"])
        else:
            s["cache"] = KV.KvCache(s["keys"].view(torch.float4_e2m1fn_x2), s["values"].view(torch.float4_e2m1fn_x2),
                                    s["key_scales"].view(torch.float8_e8m0fnu), s["value_scales"].view(torch.float8_e8m0fnu))
    cache = s["cache"]
    if op == "rotate":
        q = KV.append_rotated(cache, s["q"], s["k"], s["v"], s["positions"], s["slots"], frequencies=s["frequencies"],
                              q_weight=s["q_weight"], k_weight=s["k_weight"], interleaved=c["pairs"] != "halves")
        return [q, cache.keys, cache.values]
    if op == "token":
        out, lse = KV.attend_token(s["q"], cache, s["table"], s["lengths"], max_length=s["max_length"],
                                   sinks=c["sinks"], window=s["window"], weights=s["weights"])
        return [out, lse] if s["weights"] is None else [out, lse, s["weights"]]
    if op == "prompt":
        return list(KV.attend_prompt(s["q"], s["offsets"], cache, s["table"], s["lengths"], max_new=s["max_new"],
                                     max_length=s["max_length"], sinks=c["sinks"], window=s["window"]))
    if op == "read":
        k, v = KV.read(cache, s["slots"], dtype=s["dtype"], values=c["values"])
        return [k, v] if c["values"] else [k]
    KV.append(cache, s["table"], s["starts"], s["k"], s["v"], offsets=s["offsets"], max_new=s["max_new"])
    return list(KV.read(cache, s["all"]))


# ---- the definition in 64 bits ---------------------------------------------------
def _values64(codes, scales):
    """64-bit values [..., dim] of 4-bit rows, from the bits of a code: sign, exponent, fraction."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    e, f = (c >> 1) & 3, c & 1
    v = torch.where(e == 0, f * 0.5, (1 + 0.5 * f) * torch.exp2((e - 1).double()))
    v = torch.where(c >= 8, -v, v)
    return v * torch.exp2(scales.double() - 127).repeat_interleave(32, -1)


def _nearest64(x):
    """x [n, heads, dim] as the 4-bit values nearest to it, in 64 bits."""
    g = x.double().unflatten(-1, (-1, 32))
    top = g.abs().amax(-1, keepdim=True)
    k = torch.floor(torch.log2(torch.where(top > 0, top, 1.0)))
    k = k - (torch.exp2(k) > top).double() + (torch.exp2(k + 1) <= top).double()
    up = (top >= 1.75 * torch.exp2(k)).double()
    unit = torch.exp2(torch.where(top > 0, k - 2 + up, -125.0).clamp(-125, 125))
    y = (g / unit).abs()
    grid = torch.tensor(GRID, dtype=torch.float64, device=DEV)
    far = (y.unsqueeze(-1) - grid).abs()
    least = far.amin(-1, keepdim=True)
    even = torch.arange(8, device=DEV) % 2 == 0
    pick = torch.where(far == least, torch.where(even, 1, 2), 3).argmin(-1)
    return (torch.where(g < 0, -1.0, 1.0) * grid[pick] * unit).flatten(-2)


def _row64(s, b, rows):
    """Keys and values [kv, n, dim] of sequence b's rows in 64 bits."""
    page = s["case"]["page"]
    at = s["table"][b].long()[torch.div(rows, page, rounding_mode="floor")]
    return [_values64(s[x][at, :, rows % page], s[x[:-1] + "_scales"][at, :, rows % page]).transpose(0, 1)
            for x in ("keys", "values")]


def exact(case, seed):
    op = case["op"]
    if op == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    c = s["case"]
    page = case["page"]
    if op == "read":
        p, slot = s["slots"] // page, s["slots"] % page
        return [_values64(s[x][p, :, slot], s[x[:-1] + "_scales"][p, :, slot])
                for x in (("keys", "values") if c["values"] else ("keys",))]
    if op == "rotate":
        return _rotate64(s)
    if op == "store":
        got = []
        lens, new, off = s["lengths"].tolist(), s["new"].tolist(), s["offsets"].tolist()
        for x, tokens in (("keys", s["k"]), ("values", s["v"])):
            pool = _values64(s[x], s[x[:-1] + "_scales"])
            near = _nearest64(tokens)
            for b, n in enumerate(lens):
                rows = torch.arange(n - new[b], n, device=DEV)
                pool[s["table"][b].long()[rows // page], :, rows % page] = near[off[b]: off[b + 1]]
            got.append(pool.transpose(1, 2).flatten(0, 1))
        return got
    kv, heads = c["kv"], c["heads"]
    group = heads // kv
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device=DEV)
    weights = s["weights"].double() if s["weights"] is not None else None
    lens = s["lengths"].tolist()
    off = s["offsets"].tolist() if op == "prompt" else list(range(len(lens) + 1))
    for b, n in enumerate(lens):
        rows = torch.arange(n, device=DEV)
        k, v = _row64(s, b, rows)
        for lo in range(off[b], off[b + 1], 512):
            hi = min(off[b + 1], lo + 512)
            q = s["q"][lo:hi].double().view(hi - lo, kv, group, c["dim"]).permute(1, 2, 0, 3)
            x = torch.matmul(q.reshape(kv, -1, c["dim"]), k.transpose(1, 2).contiguous()) / math.sqrt(c["dim"])
            x = x.view(kv, group, hi - lo, -1)
            pos = n - (off[b + 1] - off[b]) + torch.arange(lo - off[b], hi - off[b], device=DEV)[:, None]
            far = rows > pos
            if s["window"] is not None:
                far = far | ((rows >= c["sinks"]) & (rows <= pos - s["window"]))
            x = x.masked_fill(far, -math.inf)
            z = torch.logsumexp(x, -1)
            p = torch.exp(x - z.masked_fill(z == -math.inf, 0.0)[..., None])
            y = torch.matmul(p.view(kv, -1, n), v.contiguous()).view(kv, group, hi - lo, c["dim"])
            out[lo:hi] = y.permute(2, 0, 1, 3).reshape(hi - lo, heads, c["dim"])
            lse[lo:hi] = z.permute(2, 0, 1).reshape(hi - lo, heads)
            if weights is not None:
                weights[b, :, :n] += p.sum((1, 2))
    return [out, lse] if weights is None else [out, lse, weights]


def _rotate64(s):
    c, page = s["case"], s["case"]["page"]
    real = s["positions"] >= 0

    def turned(x, weight):
        y = x.double()
        if weight is not None:
            y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + 1e-6) * weight.double()
        r = c["rotary"]
        if r:
            i = torch.arange(r // 2, device=DEV)
            a, b = (i, i + r // 2) if c["pairs"] == "halves" else (2 * i, 2 * i + 1)
            t = torch.polar(torch.ones((), dtype=torch.float64, device=DEV),
                            s["positions"].double()[:, None] * s["frequencies"])[:, None]
            z = torch.complex(y[..., a], y[..., b]) * t
            y = y.clone()
            y[..., a], y[..., b] = z.real, z.imag
        return y

    q = turned(s["q"], s["q_weight"])
    q[~real] = 0.0
    keys, values = s["keys"].double(), s["values"].double()
    at = s["slots"][real]
    keys[at // page, :, at % page] = turned(s["k"], s["k_weight"])[real]
    values[at // page, :, at % page] = s["v"].double()[real]
    return [q, keys, values]


def work(case):
    c, op = case, case["op"]
    if op == "plan":
        new, before = _spread(c["new"], c["ragged"], c["batch"]), _spread(c["before"], c["ragged"], c["batch"])
        # lengths, held, new, offsets, granted and the pages at hand; a token's position, sequence and slot
        pages = sum(-(-n // c["page"]) for n in new) + int(c["ends"] * sum(-(-n // c["page"]) for n in before))
        return {"bytes": 4 * 8 * c["batch"] + 8 * pages + 16 * sum(new), "flops": 0}
    dim, kv = c["dim"], c["kv"]
    row = 2 * kv * (dim // 2 + dim // 32)  # one row's 4-bit keys and values of all heads
    if op == "rotate":
        n = c["tokens"]
        return {"bytes": n * (2 * 2 * dim * (c["heads"] + 2 * kv) + 12) + 4 * c["rotary"], "flops": 0}
    if op == "read":
        half = 1 if c["values"] else 2
        return {"bytes": c["rows"] * (row // half + kv * dim * (4 if c["f32"] else 2) * 2 // half + 8), "flops": 0}
    new, rows = _new_and_all(c)
    per = -(-max(rows) // c["page"])
    if op == "store":  # new rows are read and stored, all are read back
        pool = (c["batch"] * per + 3) * c["page"]
        return {"bytes": sum(new) * (4 * kv * dim + row) + pool * (row + 4 * kv * dim + 8), "flops": 0}
    table = sum(4 * -(-n // c["page"]) for n in rows)
    q = sum(new) * c["heads"] * (2 * dim * 2 + 4)
    first, last = (c["sinks"], c["window"]) if c["window"] >= 0 else (0, max(rows))
    if op == "token":
        seen = [min(n, first + last) for n in rows]
        return {"bytes": sum(seen) * row + q + table + (8 * kv * sum(seen) if c["weights"] else 0),
                "flops": 4 * dim * c["heads"] * sum(seen)}
    pairs = 0
    for n, m in zip(new, rows):
        # rows that the last n of m queries see: up to first + last, one more for each query until then
        whole = min(max(0, m - max(first + last, m - n)), n)
        short = n - whole
        lo = m - n + 1
        pairs += short * lo + short * (short - 1) // 2 + whole * (first + last)
    reads = sum(min(m, first + last + n) for n, m in zip(new, rows))
    return {"bytes": reads * row + q + table, "flops": 4 * dim * c["heads"] * pairs}
