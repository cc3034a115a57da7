"""Serving steps as a program runs them: plan, rotated append, attention, eviction, over caches of every type."""
import math

import numpy as np
import pytest
import torch

from gpu_helpers import require_gpu
from kv4_reference import mx4_rule, mx4_values, pack
from kv_reference import attend, close
from shear_amd import kvcache as KV
from shear_amd import retrieval as R
from test_gpu_kvcache import BF16, F16, SQ8, kept_rows, normal

pytestmark = pytest.mark.gpu

HEADS, KV_HEADS, DIM, PAGE, PAGES, COLUMNS = 6, 2, 64, 16, 48, 12


@pytest.fixture(scope="module")
def gpu():
    return require_gpu()


class Server:
    """Sequences over one pool of pages, and the rows that each should hold (host, 64 bits)."""

    def __init__(self, batch, kind, q_type, seed):
        self.g = np.random.default_rng(seed)
        self.batch, self.kind, self.q_type = batch, kind, q_type
        self.cache = KV.KvCache.allocate(PAGES, KV_HEADS, PAGE, DIM, kind)
        self.shadow = KV.KvCache.allocate(PAGES, KV_HEADS, PAGE, DIM, q_type)  # the rounded rows, at the same slots

        def ints(*shape, fill=0):
            return torch.full(shape, fill, dtype=torch.int32, device="cuda")

        self.table, self.lengths, self.held = ints(batch, COLUMNS, fill=-1), ints(batch), ints(batch)
        self.free = torch.from_numpy(self.g.permutation(PAGES).astype(np.int32)).cuda()
        self.count = ints(1, fill=PAGES)
        self.frequencies = KV.rotation_frequencies(DIM)
        self.weight = normal(self.g, DIM, dtype=q_type)
        self.rows = [(np.zeros((0, KV_HEADS, DIM)), np.zeros((0, KV_HEADS, DIM))) for _ in range(batch)]

    def values(self, x):
        """Rows of the queries' type as the cache holds them."""
        x = x.double().cpu().numpy()
        if self.kind == KV.MX4:
            code, e = mx4_rule(x)
            return mx4_values(pack(code), e)
        if self.kind == SQ8:
            top = np.abs(x).max(-1, keepdims=True).astype(np.float32)
            scale = np.where(top > 0, top * np.float32(1 / 127), np.float32(1))
            y = (x.astype(np.float32) / scale).astype(np.float64)
            return np.copysign(np.floor(np.abs(y) + 0.5), y) * scale.astype(np.float64)
        return x

    def step(self, new):
        """One step; returns (queries, their attention, log-sums, plan)."""
        tokens = int(sum(max(n, 0) for n in new))
        q, k, v = (normal(self.g, tokens, h, DIM, dtype=self.q_type) for h in (HEADS, KV_HEADS, KV_HEADS))
        fresh = torch.tensor(new, dtype=torch.int32, device="cuda")
        p = KV.plan(PAGE, self.table, self.lengths, self.held, fresh, self.free, self.count, tokens)
        args = (p.positions, p.slots, self.frequencies, self.weight, self.weight)
        q = KV.append_rotated(self.cache, q, k, v, *args)
        KV.append_rotated(self.shadow, q, k, v, *args)
        self.lengths, self.held, self.count = p.lengths, p.held, p.count
        if max(new) == 1:  # one token or none: those that have one
            out, lse = KV.attend_token(*self._of_all(q, p), self.cache, self.table, p.lengths)
            of = p.sequences.long()
            out, lse = out[of], lse[of]
        else:
            out, lse = KV.attend_prompt(q, p.offsets, self.cache, self.table, p.lengths)
        granted, offsets, slots = p.granted.tolist(), p.offsets.tolist(), p.slots
        for b, n in enumerate(new):
            if n < 0:
                self.rows[b] = (np.zeros((0, KV_HEADS, DIM)), np.zeros((0, KV_HEADS, DIM)))
            at = slots[offsets[b]: offsets[b] + granted[b]]
            got = KV.read(self.shadow, at)
            self.rows[b] = tuple(np.concatenate([x, self.values(y)]) for x, y in zip(self.rows[b], got))
        return q, out, lse, p

    def _of_all(self, q, p):
        """A query for each sequence (zeros for those without a token)."""
        every = torch.zeros((self.batch, HEADS, DIM), dtype=self.q_type, device="cuda")
        every[p.sequences.long()] = q
        return (every,)

    def check(self, q, out, lse, p, new, once_more):
        assert p.lengths.tolist() == [len(k) for k, _ in self.rows]
        qh, oh, lh = (x.double().cpu().numpy() for x in (q, out, lse))
        offsets, granted = p.offsets.tolist(), p.granted.tolist()
        for b in range(self.batch):
            k, v = self.rows[b]
            for i in range(granted[b]):
                t = offsets[b] + i
                seen = np.arange(len(k)) <= len(k) - granted[b] + i
                for h in range(HEADS):
                    kh = h // (HEADS // KV_HEADS)
                    want, z, _, spread, delta = attend(qh[t, h], k[:, kh], v[:, kh], seen, 1 / math.sqrt(DIM))
                    assert close(oh[t, h], want, spread, delta, self.q_type, once_more).all(), (b, i, h)
                    assert abs(lh[t, h] - z) <= delta + 2.0**-21 * (abs(z) + 1), (b, i, h)

    def pages(self):
        """No page is in two places."""
        held, table = self.held.tolist(), self.table.cpu().numpy()
        own = [table[b, :n] for b, n in enumerate(held)] + [self.free[: int(self.count)].cpu().numpy()]
        assert np.array_equal(np.sort(np.concatenate(own)), np.arange(PAGES))
        for n, rows in zip(held, self.lengths.tolist()):
            assert n * PAGE >= rows


@pytest.mark.parametrize("kind,q_type", [(KV.MX4, BF16), (KV.MX4, F16), (SQ8, BF16), (BF16, BF16), (F16, F16)])
def test_steps(gpu, kind, q_type):
    s = Server(5, kind, q_type, 11)
    steps = [[40, 7, 0, 16, 1], [1, 1, 33, 1, 1], [1, 1, 1, 1, 1], [1, -1, 1, 1, 0], [1, 100, 1, 0, 90], [1, 1, 1, 1, 1],
             "evict", [1, 1, 1, 1, 1], [50, 1, -1, 1, 1], [0, 0, 130, 0, 150], [1, 1, 1, 1, 1]]
    for step in steps:
        if step == "evict":
            n = [len(k) for k, _ in s.rows]
            w = torch.rand((s.batch, KV_HEADS, COLUMNS * PAGE), device="cuda")
            kept, s.lengths, _ = KV.evict(s.cache, s.table, s.lengths, w, 30, sinks=2, recent=5)
            for b in range(s.batch):
                was = s.rows[b]
                rows = [kept_rows(w[b, h].cpu().numpy(), n[b], 30, 2, 5) for h in range(KV_HEADS)]
                s.rows[b] = tuple(np.stack([x[r, h] for h, r in enumerate(rows)], 1) for x in was)
            continue
        q, out, lse, p = s.step(step)
        s.check(q, out, lse, p, step, max(step) != 1)
        s.pages()
    assert p.granted.tolist() == [1] * 5


def test_a_prompt_without_pages_waits(gpu):
    s = Server(3, KV.MX4, BF16, 3)
    s.step([190, 190, 190])
    q, out, lse, p = s.step([1, 150, 1])  # 36 + 3 pages are held of 48; the second passes its table
    assert p.granted.tolist() == [1, 0, 1]
    s.pages()
    t = Server(4, KV.MX4, BF16, 4)
    t.step([190, 190, 190, 0])
    q, out, lse, p = t.step([1, 1, 1, 192])  # 12 pages are free and needed, but the first three need none: it gets them
    assert p.granted.tolist() == [1, 1, 1, 192] and int(p.count) == 0
    q, out, lse, p = t.step([5, -1, 1, 0])
    assert p.granted.tolist() == [0, 0, 1, 0]  # (the first would pass its table)
    t.pages()


@pytest.mark.parametrize("kind,q_type", [(KV.MX4, BF16), (SQ8, F16), (BF16, BF16)])
def test_a_captured_step(gpu, kind, q_type):
    """A step of single tokens in a graph, its state kept in place, replayed between eager work of the same kind."""
    s = Server(4, kind, q_type, 21)
    s.step([20, 45, 3, 31])
    g = np.random.default_rng(5)
    q, k, v = (normal(g, 4, h, DIM, dtype=q_type) for h in (HEADS, KV_HEADS, KV_HEADS))
    new = torch.ones(4, dtype=torch.int32, device="cuda")
    state = [s.table, s.lengths.clone(), s.held.clone(), s.free, s.count.clone()]

    def step(table, lengths, held, free, count, cache):
        p = KV.plan(PAGE, table, lengths, held, new, free, count, 4)
        rotated = KV.append_rotated(cache, q, k, v, p.positions, p.slots, s.frequencies, s.weight, s.weight)
        out, lse = KV.attend_token(rotated, cache, table, p.lengths, max_length=COLUMNS * PAGE)
        lengths.copy_(p.lengths)
        held.copy_(p.held)
        count.copy_(p.count)
        return out, lse

    def copied(c):
        return KV.KvCache(*(None if t is None else t.clone() for t in c._tensors()))

    other, other_cache = [x.clone() for x in state], copied(s.cache)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out, lse = step(*state, s.cache)
    for rep in range(20):  # pages begin on the way
        for x in (q, k, v):
            x.copy_(normal(np.random.default_rng(rep), *x.shape, dtype=q_type))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = step(*other, other_cache)
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1]), rep
        for a, b in zip(state, other):
            assert torch.equal(a, b), rep
    assert state[1].tolist() == [40, 65, 23, 51]


def test_a_long_context_in_4_bits(gpu):
    """Graphs over 4-bit keys, attention over what they find, eviction, all on one cache."""
    got = R.run(rows=3000, tokens=4, keep=600, dtype=KV.MX4)
    assert got["finite"] and got["lengths"] == [604, 604] and got["kept"] == 600
    # what the search finds among the 4-bit keys carries most of the attention over them, as among others
    assert got["carried"] > 0.5
