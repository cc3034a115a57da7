"""Attention over a long context through a graph index of its keys.

A prompt's keys and values go into a paged cache (``kvcache``); a graph over
each head's keys, built by ``pipeline.build_graph``, finds the rows with the
largest products with a new token's queries, and the token attends over them, the
first and the last rows.  The attention that every row gathers is kept, so that
``evict`` can shrink the cache to the rows that matter.

The graph searches by L2 distance.  A key k becomes the point (k, sqrt(M^2 -
|k|^2)) with M the largest norm, a query q the point (q, 0): then |point - query|^2
= M^2 + |q|^2 - 2 q . k, and the nearest points are the largest products.

``python -m shear_amd.retrieval`` runs a small context end to end and prints
how much of the full attention's weight the visible rows carry.
"""
from __future__ import annotations

import json
import sys
from dataclasses import dataclass, field

import torch

from . import graph as G
from . import kvcache as KV
from . import pipeline as P


class KeyIndex:
    """Graph over the keys [n, dim] of one head of one sequence."""

    def __init__(self, keys: torch.Tensor, params: P.GraphBuildParams | None = None):
        # normal keys have no clusters to speak of: larger leaves, more replication and a higher degree than the
        # builds' defaults (3,000 x 64, search lists of 100: recall@10 0.93 against 0.84, 3.7 ms against 3.4)
        if keys.shape[0] == 0:
            raise ValueError("no keys to index")
        p = params or P.GraphBuildParams(c_max=2048, fanout_top=3, fanout_second=3, l_max=96)
        k = keys.float()
        squares = (k * k).sum(1)
        last = (squares.max() - squares).clamp_(min=0.0).sqrt_()
        self.points = torch.cat([k, last[:, None]], 1).contiguous()
        n, dim = self.points.shape
        planes = torch.from_numpy(P.sketch_planes(dim, p.m_hash_bits, p.random_seed)).to(k.device)
        leaders = P.d0_leader_rows(n, P.d0_leader_count(n, dim, p), p.random_seed)
        self.graph = P.build_graph(self.points, (self.points @ planes.t()).contiguous(), leaders, p)

    def search(self, queries: torch.Tensor, count: int, list_size: int) -> torch.Tensor:
        """Rows with the largest products, int32 [queries, count], -1 where the search found fewer."""
        q = torch.nn.functional.pad(queries.float(), (0, 1))
        return G.greedy_search(self.points, self.graph.targets, self.graph.counts, self.graph.start, q,
                               max(list_size, count), count)[0]


def distinct(rows: torch.Tensor) -> torch.Tensor:
    """Row lists [..., n] in ascending order with each row once, -1 in the place of repeats."""
    s = rows.sort(-1).values
    return torch.where(torch.nn.functional.pad(s[..., 1:] == s[..., :-1], (1, 0)), -1, s)


@dataclass
class LongContext:
    """Conversations over one layer's cache: ``heads`` key heads shared by the query heads.

    The graphs cover the rows that were cached when ``build`` was called; rows added since stay
    visible until it is called again.  ``lengths`` is kept by the methods, as are the rows' counts on the
    host; a call that would pass ``max_rows`` is refused and changes nothing.  ``weights`` gathers what
    single tokens attend to (a prompt's own attention is not in it)."""

    batch: int
    heads: int
    head_dim: int
    max_rows: int                       # of a sequence, prompt and answer together
    page_rows: int = 64
    dtype: torch.dtype = torch.bfloat16  # of the cache; torch.int8: SQ8 rows
    sinks: int = 4                      # first rows that stay visible
    window: int = 256                   # last rows that stay visible
    found: int = 64                     # rows that each query head's search adds
    list_size: int = 128                # of the search
    indexes: list = field(init=False, default_factory=list)
    _rows: list = field(init=False, repr=False)     # of each sequence
    _indexed: list = field(init=False, repr=False)  # of them, in the graphs

    def __post_init__(self):
        self._rows = [0] * self.batch
        self._indexed = [0] * self.batch
        columns = -(-self.max_rows // self.page_rows)
        pages = self.batch * columns
        self.cache = KV.KvCache.allocate(pages, self.heads, self.page_rows, self.head_dim, self.dtype)
        self.table = torch.arange(pages, dtype=torch.int32, device="cuda").view(self.batch, columns)
        self.lengths = torch.zeros(self.batch, dtype=torch.int32, device="cuda")
        self.weights = torch.zeros((self.batch, self.heads, columns * self.page_rows), device="cuda")

    def _grown(self, new: list[int]) -> list[int]:
        """Rows of each sequence with ``new`` more."""
        if len(new) != self.batch or min(new, default=0) < 0:
            raise ValueError(f"new rows {new} for {self.batch} sequences")
        rows = [n + more for n, more in zip(self._rows, new)]
        if max(rows, default=0) > self.max_rows:
            raise ValueError(f"{max(rows)} rows of a sequence, room for {self.max_rows}")
        return rows

    def shown(self) -> int | None:
        """Last rows that a token sees besides the first and the found ones: ``window``, and all
        that are in no graph yet.  None: there are no graphs, every row is visible."""
        if not self.indexes:
            return None
        return max(self.window, *(n - indexed for n, indexed in zip(self._rows, self._indexed)))

    def prompt(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, new: list[int]) -> torch.Tensor:
        """Appends ``new[b]`` tokens of each sequence and returns their causal attention over all rows."""
        rows = self._grown(new)
        if sum(new) != k.shape[0]:
            raise ValueError(f"{k.shape[0]} tokens, {sum(new)} new rows")
        offsets = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device="cuda")
        KV.append(self.cache, self.table, self.lengths, k, v, offsets=offsets, max_new=max(new))
        self.lengths = self.lengths + (offsets[1:] - offsets[:-1])
        self._rows = rows
        return KV.attend_prompt(q, offsets, self.cache, self.table, self.lengths, max_new=max(new))[0]

    def build(self) -> None:
        """Graphs over the rows that are cached now."""
        self.indexes = []
        self._indexed = list(self._rows)
        for b, n in enumerate(self._rows):
            rows = torch.arange(n, device="cuda")
            pages, slots = self.table[b, rows // self.page_rows].long(), rows % self.page_rows
            keys = self.cache.keys[pages, :, slots].float()
            if self.cache.key_scales is not None:
                keys *= self.cache.key_scales[pages, :, slots].unsqueeze(-1)
            self.indexes.append([KeyIndex(keys[:, h]) for h in range(self.heads)])

    def find(self, q: torch.Tensor) -> torch.Tensor | None:
        """Rows for each sequence and key head, int32 [batch, heads, group * found], from the graphs."""
        if not self.indexes:
            return None
        group = q.shape[1] // self.heads
        rows = [[index.search(q[b, h * group: (h + 1) * group], self.found, self.list_size).flatten()
                 for h, index in enumerate(heads)] for b, heads in enumerate(self.indexes)]
        return distinct(torch.stack([torch.stack(r) for r in rows]))

    def token(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
        """Appends one token to each sequence and returns its attention over the first, the last (``shown``)
        and the found rows (over all rows while there are no graphs)."""
        rows = self._grown([1] * self.batch)
        KV.append(self.cache, self.table, self.lengths, k, v)
        self.lengths = self.lengths + 1
        self._rows = rows
        listed = self.find(q)
        return KV.attend_token(q, self.cache, self.table, self.lengths, sinks=self.sinks,
                               window=self.shown(), listed=listed, weights=self.weights)[0]

    def evict(self, keep: int) -> torch.Tensor:
        """Keeps the first, the last and the most attended rows, ``keep`` of each head, in place; the
        graphs' rows are gone, so attention is over all that is left until ``build`` is called."""
        kept, self.lengths, self.weights = KV.evict(self.cache, self.table, self.lengths, self.weights, keep,
                                                    sinks=self.sinks, recent=min(self.window, keep - self.sinks))
        self._rows = [min(n, keep) for n in self._rows]
        self.indexes = []
        return kept


def run(rows: int = 6000, batch: int = 2, heads: int = 2, group: int = 4, dim: int = 64, tokens: int = 8,
        keep: int = 1000, seed: int = 0, dtype: torch.dtype = torch.bfloat16) -> dict:
    """A context of ``rows`` rows a sequence, ``tokens`` steps with graphs, an eviction, as many steps without."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    # keys around topics; queries near the keys of some topic, so that few rows carry the attention
    topics = normal(heads, 64, dim)
    of = torch.randint(0, 64, (batch * rows, heads), generator=g, device="cuda")
    k = topics[torch.arange(heads, device="cuda"), of] + 0.4 * normal(batch * rows, heads, dim)
    v = normal(batch * rows, heads, dim)

    def queries(n):
        t = torch.randint(0, 64, (n, heads * group), generator=g, device="cuda")
        h = torch.arange(heads, device="cuda").repeat_interleave(group)
        return (topics[h, t] + 0.3 * normal(n, heads * group, dim)).bfloat16()

    c = LongContext(batch, heads, dim, rows + 2 * tokens, dtype=dtype)
    c.prompt(queries(batch * rows), k.bfloat16(), v.bfloat16(), [rows] * batch)
    c.build()
    carried = error = 0.0
    for _ in range(tokens):
        q = queries(batch)
        out = c.token(q, normal(batch, heads, dim).bfloat16(), normal(batch, heads, dim).bfloat16())
        full, lse = KV.attend_token(q, c.cache, c.table, c.lengths)
        _, seen = KV.attend_token(q, c.cache, c.table, c.lengths, sinks=c.sinks, window=c.shown(), listed=c.find(q))
        carried += float(torch.exp(seen - lse).mean()) / tokens
        error += float((out.float() - full.float()).norm() / full.float().norm()) / tokens
    kept = c.evict(keep)
    for _ in range(tokens):
        out = c.token(queries(batch), normal(batch, heads, dim).bfloat16(), normal(batch, heads, dim).bfloat16())
    return {"rows": rows, "visible": c.sinks + c.window + group * c.found, "carried": carried, "error": error,
            "kept": int((kept >= 0).sum()) // (batch * heads), "lengths": c.lengths.tolist(),
            "finite": bool(out.isfinite().all())}


if __name__ == "__main__":
    print(json.dumps(run(*(int(a) for a in sys.argv[1:]))))
