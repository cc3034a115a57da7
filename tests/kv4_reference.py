"""Plain forms of the key-value cache's 4-bit rows, of the plan of a step and of the rotated append, for the tests:
loops and 64 bits, straight from the formulas."""
from __future__ import annotations

import numpy as np
import torch

from shear_amd import kvcache as KV

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def mx4_rule(x):
    """(codes uint8 [..., dim], scale bytes uint8 [..., dim / 32]) of rows of finite or other f64 values."""
    g = np.asarray(x, np.float64).reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    with np.errstate(all="ignore"):
        top = np.abs(g).max(-1)
        finite = np.isfinite(g).all(-1)
        m, k = np.frexp(np.where(finite, top, 0.0))  # m in [0.5, 1)
        e = np.where(top > 0, k - 1 - 2 + (m >= 0.875) + 127, 0).clip(2, 252)
        y = np.where(finite[..., None], g, 0.0) / np.exp2(e.astype(np.float64) - 127)[..., None]
        far = np.abs(np.abs(y)[..., None] - GRID)
    least = far.min(-1, keepdims=True)
    # the nearest, of two the even code
    code = np.where(far == least, np.arange(8) % 2, 2).argmin(-1)
    code = code + 8 * np.signbit(y)
    code[~finite] = 0
    e[~finite] = 255
    return code.reshape(x.shape).astype(np.uint8), e.astype(np.uint8)


def mx4_values(packed, scales):
    """f64 [..., dim] of bytes of two codes and scale bytes (255: NaN)."""
    code = np.stack([packed & 15, packed >> 4], -1).reshape(*packed.shape[:-1], 2 * packed.shape[-1])
    v = GRID[code & 7] * np.where(code >= 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return v * np.repeat(s, 32, -1)


def pack(code):
    return code[..., 0::2] | code[..., 1::2] << 4


class Pool4:
    """A 4-bit cache whose unused slots are NaN, with a random page table (as ``kv_reference.Pool``)."""

    def __init__(self, batch, columns, heads, page_rows, dim, seed, spare=3, transposed=False, apart=0):
        g = np.random.default_rng(seed)
        pages = batch * columns + spare
        shape = (pages, page_rows, heads) if transposed else (pages, heads, page_rows)

        def pool(width, fill, dtype):
            t = torch.full((*shape, width + apart), fill, dtype=torch.uint8, device="cuda")[..., :width]
            return (t.transpose(1, 2) if transposed else t).view(dtype)

        self.cache = KV.KvCache(*(self._rows(shape, dim // 2, transposed) for _ in range(2)),
                                *(pool(dim // 32, 255, torch.float8_e8m0fnu) for _ in range(2)))
        self.table_host = g.permutation(pages)[: batch * columns].reshape(batch, columns).astype(np.int32)
        self.table = torch.from_numpy(self.table_host).cuda()
        self.page_rows = page_rows

    @staticmethod
    def _rows(shape, width, transposed):
        t = torch.full((*shape, width), 0x77, dtype=torch.uint8, device="cuda")
        return (t.transpose(1, 2) if transposed else t).view(KV.MX4)

    def bytes(self):
        """(keys, values, key scales, value scales) as bytes on the host, and their tensors as bytes."""
        c = self.cache
        return [t.view(torch.uint8) for t in (c.keys, c.values, c.key_scales, c.value_scales)]

    def fill(self, lengths, k, v):
        """Rows 0..lengths[b] of each sequence from k, v [sum of lengths, heads, dim], written by the rule."""
        at = 0
        for b, n in enumerate(lengths):
            self.put(self.table_host[b], np.arange(n), k[at: at + n], v[at: at + n])
            at += n

    def put(self, table, rows, k, v):
        if not len(rows):
            return
        page = torch.from_numpy(table[rows // self.page_rows].astype(np.int64)).cuda()
        slot = torch.from_numpy(rows % self.page_rows).cuda()
        kc, vc, ks, vs = self.bytes()
        for x, codes, scales in ((k, kc, ks), (v, vc, vs)):
            code, e = mx4_rule(x.double().cpu().numpy())
            codes[page, :, slot] = torch.from_numpy(pack(code)).cuda()
            scales[page, :, slot] = torch.from_numpy(e).cuda()

    def rows(self, b, n, head):
        """(keys, values) f64 [n, dim] as the cache holds them, and which rows have a page."""
        j = np.arange(n)
        page = self.table_host[b][j // self.page_rows].astype(np.int64)
        there = (page >= 0) & (page < self.cache.keys.shape[0])
        at, slot = torch.from_numpy(np.where(there, page, 0)).cuda(), torch.from_numpy(j % self.page_rows).cuda()
        kc, vc, ks, vs = self.bytes()
        return (*(mx4_values(c[at, head, slot].cpu().numpy(), s[at, head, slot].cpu().numpy())
                  for c, s in ((kc, ks), (vc, vs))), there)


def plan(page_rows, table, lengths, held, new, free, count, tokens):
    """``kvcache.plan`` on the host: (lengths, held, count, granted, offsets, positions, sequences, slots, table, free)."""
    table, free = table.copy(), free.copy()
    batch, columns = table.shape
    covers = min(columns * page_rows, 2**30 - 1)
    offsets, top = [0], min(max(int(count), 0), len(free))
    grow, target = [], []
    for b in range(batch):
        n, rows, has = max(int(new[b]), 0), min(max(int(lengths[b]), 0), covers), min(max(int(held[b]), 0), columns)
        offsets.append(offsets[-1] + n)
        fits = rows + n <= covers and offsets[-1] <= tokens
        grow.append(n if fits else 0)
        target.append(0 if new[b] < 0 else -(-(rows + grow[-1]) // page_rows))
        for c in range(target[-1], has):
            if top < len(free):
                free[top] = table[b, c]
            top += 1
    after, own, granted = [], [], []
    need, left = 0, top
    positions, sequences, slots = (np.full(tokens, -1, np.int64) for _ in range(3))
    for b in range(batch):
        rows, has = min(max(int(lengths[b]), 0), covers), min(max(int(held[b]), 0), columns)
        more = max(0, target[b] - has)
        need += more
        served = more == 0 or need <= top
        if served:
            for c in range(has, target[b]):
                left -= 1
                table[b, c] = free[left] if left < len(free) else -1
        granted.append(grow[b] if served else 0)
        own.append(target[b] if served else has)
        after.append(0 if new[b] < 0 else rows + granted[-1])
        for i in range(offsets[b], min(offsets[b + 1], tokens)):
            sequences[i] = b
            at = i - offsets[b]
            if at < granted[-1]:
                row = rows + at
                positions[i] = row
                page = int(table[b, row // page_rows])
                slots[i] = page * page_rows + row % page_rows if page >= 0 else -1
    return after, own, [min(left, len(free))], granted, offsets, positions, sequences, slots, table, free


def rotated(x, positions, frequencies, weight, eps, interleaved):
    """(y f64, size) of x [tokens, heads, dim] f64: the normalized and rotated rows, and the size that an error of one unit in
    the last place has for each value (the pair's values before the rotation)."""
    y = x.copy()
    if weight is not None:
        y = y / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight
    size = np.abs(y)
    if frequencies is not None and len(frequencies):
        r = 2 * len(frequencies)
        i = np.arange(r // 2)
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
        t = (positions.astype(np.longdouble)[:, None] * frequencies.astype(np.longdouble)).astype(np.longdouble)
        cos, sin = np.cos(t).astype(np.float64)[:, None], np.sin(t).astype(np.float64)[:, None]
        ya, yb = y[..., a].copy(), y[..., b].copy()
        y[..., a], y[..., b] = ya * cos - yb * sin, ya * sin + yb * cos
        both = np.abs(ya) + np.abs(yb)
        size[..., a] = size[..., b] = both
    return y, size
