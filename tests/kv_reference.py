"""Plain 64-bit forms of the key-value cache's operators, for the GPU tests:
loops over sequences and heads, straight from the formulas, on host copies."""
from __future__ import annotations

import math

import numpy as np
import torch

from shear_amd import kvcache as KV

# largest relative error of one rounding to the type
ROUND = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


class Pool:
    """A cache whose unused slots hold NaN (SQ8: NaN scales), with a random page table."""

    def __init__(self, batch, columns, heads, page_rows, dim, dtype, seed, spare=3, transposed=False):
        g = np.random.default_rng(seed)
        pages = batch * columns + spare
        shape = (pages, page_rows, heads, dim) if transposed else (pages, heads, page_rows, dim)

        def pool(shape, dtype):
            t = torch.zeros(shape, dtype=dtype, device="cuda")
            if dtype != torch.int8:
                t.fill_(float("nan"))
            return t.transpose(1, 2) if transposed else t

        scales = [pool(shape[:3], torch.float32) for _ in range(2)] if dtype == torch.int8 else [None, None]
        self.cache = KV.KvCache(pool(shape, dtype), pool(shape, dtype), *scales)
        self.table_host = g.permutation(pages)[: batch * columns].reshape(batch, columns).astype(np.int32)
        self.table = torch.from_numpy(self.table_host).cuda()
        self.page_rows = page_rows

    def fill(self, lengths, k, v):
        """Rows 0..lengths[b] of each sequence from k, v [sum of lengths, heads, dim] (device)."""
        off = torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32, device="cuda")
        start = torch.zeros(len(lengths), dtype=torch.int32, device="cuda")
        KV.append(self.cache, self.table, start, k, v, offsets=off, max_new=int(max(lengths)))

    def rows(self, b, n, head):
        """(keys, values) f64 [n, dim] as the cache holds them, NaN where a page id names no page."""
        c = self.cache
        j = np.arange(n)
        page = torch.from_numpy(self.table_host[b][j // self.page_rows].astype(np.int64))
        there = (page >= 0) & (page < c.keys.shape[0])
        at, slot = torch.where(there, page, 0).cuda(), torch.from_numpy(j % self.page_rows).cuda()
        out = []
        for x, s in ((c.keys, c.key_scales), (c.values, c.value_scales)):
            y = x[at, head, slot].double()
            if s is not None:
                y = y * s[at, head, slot].double()[:, None]
            out.append(y.cpu().numpy())
        return out[0], out[1], there.numpy()


def attend(q, k, v, seen, scale):
    """(out [dim], lse, p [n], spread, delta): one query in 64 bits over the rows that
    ``seen`` marks.  spread = sum p |v| and delta, a bound on the error that f32
    arithmetic of length dim puts into a logit, are what tolerances are made of."""
    out, p = np.zeros(v.shape[1]), np.zeros(len(k))
    idx = np.nonzero(seen)[0]
    if len(idx) == 0:
        return out, -math.inf, p, out, 0.0
    with np.errstate(all="ignore"):
        x = (k[idx] @ q) * scale
        delta = float((np.abs(k[idx]) @ np.abs(q)).max()) * scale * (len(q) + 8) * 2.0**-24
        real = x > -np.inf
        real |= np.isnan(x)
        if not real.any():
            return out, -math.inf, p, out, 0.0
        m = x[real].max()
        e = np.where(real, np.exp(x - m), 0.0)
        total = e.sum()
        p[idx] = e / total
        vv = v[idx][real]
        pr = p[idx][real][:, None]
        return (pr * vv).sum(0), float(m + np.log(total)), p, (pr * np.abs(vv)).sum(0), delta


def close(got, want, spread, delta, dtype, once_more):
    """Whether an output row is within one rounding of the result, a relative error
    of the weights (the logits' errors in numerator and sum, f32 exponentials and
    sums) and, where the kernel rounds the weights, one rounding of each."""
    u = ROUND[dtype]
    # results below f32's smallest normal number are no numbers of either type
    tol = 2.0**-126 + u * np.abs(want) + (2 * delta + 2.0**-19 + (u if once_more else 0.0)) * spread
    if dtype == torch.float16:
        tol = tol + 2.0**-24 + (2.0**-24 if once_more else 0.0) * spread.max(initial=0.0)
    return np.abs(got - want) <= tol * 1.01
