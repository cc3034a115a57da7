"""Performance cases of the paged key-value cache: append, attention of single
tokens and of prompts, eviction.

Each case is one call of one of the four operators (``op``) at the sizes it
gives.  With ``own`` false a pass computes the operator with elementary torch
operations in 32 bits; with ``own`` true it calls the package.  Lengths of the
sequences of one case are spread between ``ragged`` times the case's length and
the whole of it, in an order that the seed draws, so the work is a function of
the case alone.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # One conversation near its start, few narrow heads: launch and latency.
        {"name": "token_small", "op": "token", "batch": 1, "heads": 8, "kv": 2, "dim": 64, "rows": 201, "ragged": 1.0,
         "type": "bf16", "sq8": False, "page": 16, "sinks": 0, "window": -1, "found": 0, "weights": False},
        # A served batch at mid length, accumulating the weights that eviction goes by.
        {"name": "token_batch", "op": "token", "batch": 48, "heads": 32, "kv": 8, "dim": 128, "rows": 4100,
         "ragged": 0.3, "type": "bf16", "sq8": False, "page": 32, "sinks": 0, "window": -1, "found": 0,
         "weights": True},
        # One long document: only the split over its length fills the card.
        {"name": "token_long", "op": "token", "batch": 1, "heads": 32, "kv": 4, "dim": 128, "rows": 131071,
         "ragged": 1.0, "type": "f16", "sq8": False, "page": 64, "sinks": 0, "window": -1, "found": 0,
         "weights": False},
        # A batch of long documents kept in SQ8 rows.
        {"name": "token_sq8", "op": "token", "batch": 8, "heads": 32, "kv": 8, "dim": 128, "rows": 40000,
         "ragged": 0.5, "type": "bf16", "sq8": True, "page": 128, "sinks": 0, "window": -1, "found": 0,
         "weights": True},
        # Rows that a graph search found, with the first and the last rows of long documents.
        {"name": "token_found", "op": "token", "batch": 16, "heads": 16, "kv": 4, "dim": 96, "rows": 60000,
         "ragged": 0.5, "type": "bf16", "sq8": False, "page": 64, "sinks": 4, "window": 512, "found": 1500,
         "weights": False},
        # The next few words of some conversations at once.
        {"name": "prompt_small", "op": "prompt", "batch": 3, "heads": 8, "kv": 8, "dim": 64, "new": 70, "before": 130,
         "ragged": 0.2, "type": "f16", "sq8": False, "page": 16, "sinks": 0, "window": -1},
        # Whole prompts, causal.
        {"name": "prompt_causal", "op": "prompt", "batch": 2, "heads": 16, "kv": 4, "dim": 128, "new": 4096,
         "before": 0, "ragged": 1.0, "type": "bf16", "sq8": False, "page": 64, "sinks": 0, "window": -1},
        # A long prompt with a sliding window and first rows that stay visible.
        {"name": "prompt_window", "op": "prompt", "batch": 1, "heads": 16, "kv": 4, "dim": 128, "new": 12001,
         "before": 0, "ragged": 1.0, "type": "bf16", "sq8": False, "page": 64, "sinks": 4, "window": 1024},
        # A short cache cut to a small budget: latency.
        {"name": "evict_small", "op": "evict", "batch": 2, "kv": 2, "dim": 64, "rows": 700, "ragged": 0.5,
         "type": "f16", "page": 16, "keep": 256, "sinks": 4, "recent": 64},
        # A batch of long documents cut to a quarter.
        {"name": "evict_large", "op": "evict", "batch": 8, "kv": 8, "dim": 128, "rows": 32768, "ragged": 0.6,
         "type": "bf16", "page": 64, "keep": 8000, "sinks": 4, "recent": 500},
        # One new row for each sequence of a batch.
        {"name": "append_token", "op": "append", "batch": 64, "kv": 8, "dim": 128, "new": 1, "before": 1000,
         "ragged": 1.0, "type": "bf16", "sq8": False, "page": 32},
        # Prompts of a batch into an SQ8 cache.
        {"name": "append_prompt_sq8", "op": "append", "batch": 4, "kv": 8, "dim": 128, "new": 4096, "before": 0,
         "ragged": 0.5, "type": "bf16", "sq8": True, "page": 64},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng: random.Random):
    op = rng.choice(["token", "token", "token", "prompt", "prompt", "evict", "append"])
    kv = rng.choice([1, 2, 4, 8])
    dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
    c = {"op": op, "kv": kv, "dim": dim, "ragged": rng.choice([0.1, 0.5, 1.0]), "type": rng.choice(["bf16", "f16"]),
         "page": rng.choice([16, 32, 64, 128])}
    sinks, window = rng.choice([(0, -1), (0, -1), (rng.randint(0, 8), rng.randint(100, 2000))])
    if op == "token":
        c["heads"] = kv * rng.choice([1, 2, 4, 7, 8, 16])
        c["rows"] = _log(rng, 30, 131072)
        c["batch"] = _log(rng, 1, min(64, max(1.0, 8e8 / (2 * c["rows"] * kv * dim))))
        c["sq8"] = rng.random() < 0.35
        c["found"] = 0 if window < 0 else rng.choice([0, min(c["rows"], _log(rng, 50, 2500))])
        c["weights"] = rng.random() < 0.5
        c["sinks"], c["window"] = sinks, window
    elif op == "prompt":
        c["heads"] = kv * rng.choice([1, 2, 4, 8])
        c["new"] = _log(rng, 2, 8000)
        c["before"] = rng.choice([0, _log(rng, 10, 20000)])
        pairs = c["new"] * (c["before"] + c["new"])
        c["batch"] = _log(rng, 1, min(8, max(1.0, 16 * 4096 * 4096 * 2 * 128 / (pairs * c["heads"] * dim))))
        if pairs * c["heads"] * dim > 16 * 4096 * 4096 * 2 * 128:
            c["new"], c["before"] = min(c["new"], 1500), min(c["before"], 3000)
        c["sq8"] = rng.random() < 0.3
        c["sinks"], c["window"] = sinks, window
    elif op == "evict":
        c["rows"] = _log(rng, 100, 100000)
        c["batch"] = _log(rng, 1, min(32, max(1.0, 2.6e8 / (c["rows"] * kv * dim))))
        c["keep"] = max(20, int(c["rows"] * rng.uniform(0.1, 0.7)))
        c["sinks"] = rng.randint(0, 8)
        c["recent"] = rng.randint(0, c["keep"] - c["sinks"])
    else:
        c["new"] = rng.choice([1, _log(rng, 2, 4096)])
        c["before"] = rng.randint(0, 3000)
        c["batch"] = _log(rng, 1, min(64, max(1.0, 1.6e7 / (c["new"] * kv * dim))))
        c["sq8"] = rng.random() < 0.4
    return c


def _spread(most, ragged, batch):
    """Lengths from ragged * most to most, evenly spread."""
    least = max(1, int(most * ragged))
    return [most - (most - least) * b // max(1, batch - 1) for b in range(batch)]


def _new_and_all(case):
    """New rows and all rows of each sequence of a case."""
    if case["op"] in ("token", "evict"):
        rows = _spread(case["rows"], case["ragged"], case["batch"])
        return [1] * len(rows), rows
    new = _spread(case["new"], case["ragged"], case["batch"])
    return new, [n + case["before"] for n in new]


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    batch, kv, dim, page, op = case["batch"], case["kv"], case["dim"], case["page"], case["op"]
    dt = DTYPES[case["type"]]
    order = torch.randperm(batch, generator=g, device=DEV)
    new, rows = (torch.tensor(v, dtype=torch.int32, device=DEV)[order].contiguous() for v in _new_and_all(case))
    most = max(_new_and_all(case)[1])
    per = -(-most // page)
    extra = batch * -(-case["keep"] // page) if op == "evict" else 3
    pages = batch * per + extra
    ids = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    s = {"case": dict(case), "lengths": rows, "max_length": most, "table": ids[: batch * per].view(batch, per)}

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32 if len(shape) < 3 else dt)

    keys, values = normal(pages, kv, page, dim), normal(pages, kv, page, dim)
    s["key_scales"] = s["value_scales"] = None
    if case.get("sq8"):
        (keys, s["key_scales"]), (values, s["value_scales"]) = _sq8(keys), _sq8(values)
    s["keys"], s["values"] = keys, values
    if op == "token":
        s["q"] = normal(batch, case["heads"], dim) * 2
        s["window"] = None if case["window"] < 0 else case["window"]
        s["weights"] = torch.rand((batch, kv, per * page), generator=g, device=DEV) if case["weights"] else None
        s["found"] = None
        if case["found"]:  # distinct rows for each head, some of them in the window, a few places empty
            n, step = case["found"], max(1, min(_new_and_all(case)[1]) // case["found"])
            at = torch.arange(n, device=DEV) * step + torch.randint(0, step, (batch, kv, n), generator=g, device=DEV)
            at = torch.where(torch.rand(at.shape, generator=g, device=DEV) < 0.02, -1, at)
            s["found"] = at.to(torch.int32)
    elif op == "prompt":
        s["offsets"] = torch.nn.functional.pad(new.cumsum(0), (1, 0)).to(torch.int32)
        s["max_new"] = max(_new_and_all(case)[0])
        s["q"] = normal(sum(_new_and_all(case)[0]), case["heads"], dim) * 2
        s["window"] = None if case["window"] < 0 else case["window"]
    elif op == "evict":
        s["into"] = ids[batch * per:].view(batch, -1)
        w = torch.randn((batch, kv, per * page), generator=g, device=DEV).mul_(2).exp_()
        s["weights"] = torch.where(torch.rand(w.shape, generator=g, device=DEV) < 0.05, 0.0, w)
    else:
        s["starts"] = rows - new
        s["offsets"] = torch.nn.functional.pad(new.cumsum(0), (1, 0)).to(torch.int32) if case["new"] > 1 else None
        s["max_new"] = max(_new_and_all(case)[0])
        s["new"] = new
        total = sum(_new_and_all(case)[0])
        s["k"], s["v"] = normal(total, kv, dim), normal(total, kv, dim)
    return s


def _sq8(x):
    """SQ8 codes and scales of rows: the scale is max|x| / 127, the code the quotient rounded half away from zero."""
    x = x.float()
    top = x.abs().amax(-1)
    scale = torch.where(top > 0, top / 127.0, 1.0)
    q = x / scale.unsqueeze(-1)
    code = torch.floor(q.abs().double() + 0.5).clamp(max=127.0).to(torch.float32) * torch.sign(q)
    return code.to(torch.int8), scale


# ---- plain forms ---------------------------------------------------------------
def _gather(s, what, rows, head=True):
    """Rows [batch, kv, n] of the cache as f32 [batch, kv, n, dim]."""
    page = s["case"]["page"]
    b = torch.arange(rows.shape[0], device=DEV)[:, None, None]
    h = torch.arange(rows.shape[1], device=DEV)[None, :, None]
    p = s["table"][b, rows // page].long()
    x = s[what][p, h, rows % page].float()
    scales = s["key_scales"] if what == "keys" else s["value_scales"]
    return x if scales is None else x * scales[p, h, rows % page].unsqueeze(-1)


def _softmax(x, seen):
    """(p, 1 / sum p or 0, log of the sum of exp) over the last axis, of the places that `seen` marks."""
    x = torch.where(seen, x, -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(x - m)
    total = p.sum(-1, keepdim=True)
    return p, torch.where(total > 0, 1.0 / total, 0.0), (m + torch.log(total)).squeeze(-1)


def _token(s):
    c, lens = s["case"], s["lengths"].long()
    batch, kv, dim, heads = c["batch"], c["kv"], c["dim"], c["heads"]
    length = lens[:, None, None]
    if s["window"] is None:
        rows = torch.arange(s["max_length"], device=DEV).expand(batch, kv, -1)
        seen = rows < length
    else:
        first = torch.arange(c["sinks"], device=DEV).expand(batch, kv, -1)
        last = length - 1 - torch.arange(c["window"], device=DEV).expand(batch, kv, -1)
        rows = torch.cat([first, last], -1)
        seen = torch.cat([first < length, last >= c["sinks"]], -1)
        if s["found"] is not None:
            f = s["found"].long()
            rows = torch.cat([rows, f], -1)
            seen = torch.cat([seen, (f >= c["sinks"]) & (f < length - c["window"])], -1)
    rows = torch.where(seen, rows, 0)
    q = s["q"].float().view(batch, kv, heads // kv, dim)
    logits = torch.matmul(q, _gather(s, "keys", rows).transpose(-1, -2)) / math.sqrt(dim)
    p, inv, lse = _softmax(logits, seen.unsqueeze(2))
    v = torch.where(seen.unsqueeze(-1), _gather(s, "values", rows), 0.0)
    out = (torch.matmul(p, v) * inv).view(batch, heads, dim).to(s["q"].dtype)
    got = [out, lse.view(batch, heads)]
    if s["weights"] is not None:
        s["weights"].scatter_add_(2, rows, torch.where(seen, (p * inv).sum(2), 0.0))
        got.append(s["weights"])
    return got


def _prompt(s):
    c, lens = s["case"], s["lengths"].long()
    batch, kv, dim, heads, n = c["batch"], c["kv"], c["dim"], c["heads"], s["max_new"]
    off = s["offsets"].long()
    new = (off[1:] - off[:-1])[:, None]
    i = torch.arange(n, device=DEV).expand(batch, -1)
    token = torch.where(i < new, off[:-1, None] + i, 0)
    q = s["q"].float()[token].view(batch, n, kv, heads // kv, dim).permute(0, 2, 3, 1, 4)
    pos = (lens[:, None] - new + i)[:, :, None]
    j = torch.arange(s["max_length"], device=DEV)
    seen = (j <= pos) & (j < lens[:, None, None])
    if s["window"] is not None:
        seen &= (j < c["sinks"]) | (j > pos - s["window"])
    rows = torch.where(j < lens[:, None, None], j, 0).expand(batch, kv, -1)
    k, v = _gather(s, "keys", rows).unsqueeze(2), _gather(s, "values", rows).unsqueeze(2)
    p, inv, lse = _softmax(torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(dim), seen[:, None, None])
    out = (torch.matmul(p, v) * inv).permute(0, 3, 1, 2, 4).reshape(batch * n, heads, dim)
    real = (i < new).reshape(-1).nonzero().squeeze(-1)
    return [out[real].to(s["q"].dtype), lse.permute(0, 3, 1, 2).reshape(batch * n, heads)[real]]


def _evict(s):
    c, lens = s["case"], s["lengths"].long()[:, None, None]
    keep, page, batch, kv = c["keep"], c["page"], c["batch"], c["kv"]
    w = s["weights"]
    j = torch.arange(w.shape[-1], device=DEV)
    always = (j < c["sinks"]) | (j >= lens - c["recent"]) | (lens <= keep)
    rank = torch.where(j < lens, torch.where(always, math.inf, torch.where(w.isnan(), -1.0, w)), -math.inf)
    best = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    count = torch.minimum(lens, torch.tensor(keep, device=DEV))
    at = torch.arange(keep, device=DEV)
    rows = torch.sort(torch.where(at < count, best, 1 << 40), dim=-1).values
    kept = torch.where(at < count, rows, -1)
    new_weights = torch.zeros_like(w)
    new_weights[..., :keep] = torch.where(at < count, torch.gather(w, 2, kept.clamp(min=0)), 0.0)
    b, h, t = (at < count).expand(batch, kv, -1).nonzero(as_tuple=True)
    src, dst = kept[b, h, t], s["into"][b, t // page].long()
    src_page = s["table"][b, src // page].long()
    s["keys"][dst, h, t % page] = s["keys"][src_page, h, src % page]
    s["values"][dst, h, t % page] = s["values"][src_page, h, src % page]
    return [kept.to(torch.int32), count.view(-1).to(torch.int32), new_weights, s["keys"], s["values"]]


def _append(s):
    c, new = s["case"], s["new"].long()
    b = torch.repeat_interleave(torch.arange(c["batch"], device=DEV), new, output_size=s["k"].shape[0])
    first = new.cumsum(0) - new
    row = s["starts"].long()[b] + torch.arange(b.numel(), device=DEV) - first[b]
    at, slot = s["table"][b, row // c["page"]].long(), row % c["page"]
    if s["key_scales"] is None:
        s["keys"][at, :, slot], s["values"][at, :, slot] = s["k"], s["v"]
        return [s["keys"], s["values"]]
    s["keys"][at, :, slot], s["key_scales"][at, :, slot] = _sq8(s["k"])
    s["values"][at, :, slot], s["value_scales"][at, :, slot] = _sq8(s["v"])
    return [s["keys"] * s["key_scales"].unsqueeze(-1), s["values"] * s["value_scales"].unsqueeze(-1)]


def run(s):
    op, c = s["case"]["op"], s["case"]
    if not own:
        return {"token": _token, "prompt": _prompt, "evict": _evict, "append": _append}[op](s)
    from shear_amd import kvcache as KV

    if "cache" not in s:
        s["cache"] = KV.KvCache(s["keys"], s["values"], s["key_scales"], s["value_scales"])
    cache = s["cache"]
    if op == "token":
        out, lse = KV.attend_token(s["q"], cache, s["table"], s["lengths"], max_length=s["max_length"],
                                   sinks=c["sinks"], window=s["window"], listed=s["found"], weights=s["weights"])
        return [out, lse] if s["weights"] is None else [out, lse, s["weights"]]
    if op == "prompt":
        return list(KV.attend_prompt(s["q"], s["offsets"], cache, s["table"], s["lengths"], max_new=s["max_new"],
                                     max_length=s["max_length"], sinks=c["sinks"], window=s["window"]))
    if op == "evict":
        got = KV.evict(cache, s["table"], s["lengths"], s["weights"], c["keep"], sinks=c["sinks"], recent=c["recent"],
                       max_length=s["max_length"], into=s["into"])
        return [*got, cache.keys, cache.values]
    KV.append(cache, s["table"], s["starts"], s["k"], s["v"], offsets=s["offsets"], max_new=s["max_new"])
    if cache.key_scales is None:
        return [cache.keys, cache.values]
    return [cache.keys * cache.key_scales.unsqueeze(-1), cache.values * cache.value_scales.unsqueeze(-1)]


# ---- the definition in 64 bits ---------------------------------------------------
def _row64(s, b, rows):
    """Keys and values [kv, n, dim] of sequence b's rows (one list for all heads, or [kv, n]) in 64 bits."""
    page, kv = s["case"]["page"], s["case"]["kv"]
    rows = rows.expand(kv, -1)
    at = s["table"][b].long()[torch.div(rows, page, rounding_mode="floor")]
    h = torch.arange(kv, device=DEV)[:, None]
    got = []
    for x, scale in ((s["keys"], s["key_scales"]), (s["values"], s["value_scales"])):
        y = x[at, h, rows % page].double()
        got.append(y if scale is None else y * scale[at, h, rows % page].double()[..., None])
    return got


def exact(case, seed):
    if case["op"] not in ("token", "prompt"):
        return None  # rows are chosen and moved, nothing is computed
    s = prepare(case, seed)
    c, kv, heads = s["case"], case["kv"], case["heads"]
    group = heads // kv
    out, lse = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV), torch.full(s["q"].shape[:2], -math.inf,
                                                                                      dtype=torch.float64, device=DEV)
    weights = s["weights"].double() if c["op"] == "token" and s["weights"] is not None else None
    lens = s["lengths"].tolist()
    off = s["offsets"].tolist() if c["op"] == "prompt" else list(range(len(lens) + 1))
    for b, n in enumerate(lens):
        if c["op"] == "token" and s["window"] is not None:
            lists = []
            for h in range(kv):
                found = [] if s["found"] is None else [r for r in s["found"][b, h].tolist() if 0 <= r < n]
                lists.append(sorted(set(range(min(c["sinks"], n))) | set(range(max(0, n - s["window"]), n)) | set(found)))
            width = max(len(r) for r in lists)
            rows = torch.tensor([r + [0] * (width - len(r)) for r in lists], device=DEV)
            real = torch.tensor([[True] * len(r) + [False] * (width - len(r)) for r in lists], device=DEV)
        else:
            rows = torch.arange(n, device=DEV)[None]
            real = torch.ones((1, n), dtype=torch.bool, device=DEV)
        k, v = _row64(s, b, rows)
        for lo in range(off[b], off[b + 1], 512):
            hi = min(off[b + 1], lo + 512)
            q = s["q"][lo:hi].double().view(hi - lo, kv, group, c["dim"]).permute(1, 2, 0, 3)
            x = torch.matmul(q.reshape(kv, -1, c["dim"]), k.transpose(1, 2)) / math.sqrt(c["dim"])
            x = x.view(kv, group, hi - lo, -1)
            hide = ~real[:, None, None, :].expand(x.shape)
            if c["op"] == "prompt":
                pos = n - (off[b + 1] - off[b]) + torch.arange(lo - off[b], hi - off[b], device=DEV)[:, None]
                far = rows > pos
                if s["window"] is not None:
                    far = far | ((rows >= c["sinks"]) & (rows <= pos - s["window"]))
                hide = far.expand(x.shape)
            x = x.masked_fill(hide, -math.inf)
            z = torch.logsumexp(x, -1)
            p = torch.exp(x - z.masked_fill(z == -math.inf, 0.0)[..., None])
            y = torch.matmul(p.view(kv, -1, p.shape[-1]), v).view(kv, group, hi - lo, c["dim"])
            out[lo:hi] = y.permute(2, 0, 1, 3).reshape(hi - lo, heads, c["dim"])
            lse[lo:hi] = z.permute(2, 0, 1).reshape(hi - lo, heads)
            if weights is not None:
                weights[b].scatter_add_(1, rows.expand(kv, -1), p.sum((1, 2)))
    return [out, lse] if weights is None else [out, lse, weights]


def work(case):
    c, dim, kv = case, case["dim"], case["kv"]
    size = 1 if c.get("sq8") else 2
    row = 2 * kv * (dim * size + (4 if c.get("sq8") else 0))  # one row's keys and values of all heads
    new, rows = _new_and_all(c)
    table = sum(4 * -(-n // c["page"]) for n in rows)
    if c["op"] == "append":
        return {"bytes": sum(new) * (2 * kv * dim * 2 + row) + 8 * len(new), "flops": 0}
    if c["op"] == "evict":
        kept = sum(min(n, c["keep"]) for n in rows)
        most = -(-c["rows"] // c["page"]) * c["page"]
        return {"bytes": 2 * kept * row + 4 * kv * (sum(rows) + c["batch"] * (c["keep"] + most)) + 2 * table, "flops": 0}
    q = sum(new) * c["heads"] * (2 * dim * 2 + 4)
    first, last = (c["sinks"], c["window"]) if c["window"] >= 0 else (0, max(rows))
    if c["op"] == "token":
        # of the rows found, the share before the window counts
        seen = [min(n, first + last) + int(c["found"] * 0.98 * max(0.0, 1 - (first + last) / n)) for n in rows]
        seen = [min(n, m) for n, m in zip(rows, seen)]
        extra = 8 * kv * sum(seen) if c["weights"] else 0
        return {"bytes": sum(seen) * row + q + table + extra + 4 * kv * c["batch"] * c["found"],
                "flops": 4 * dim * c["heads"] * sum(seen)}
    pairs = 0
    for n, m in zip(new, rows):
        pos = np.arange(m - n, m, dtype=np.int64)
        pairs += int(np.minimum(pos + 1, np.minimum(first, np.maximum(0, pos + 1 - last)) + last).sum())
    reads = sum(m if c["window"] < 0 else min(m, first + last + n) for n, m in zip(new, rows))
    return {"bytes": reads * row + q + table, "flops": 4 * dim * c["heads"] * pairs}
