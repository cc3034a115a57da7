"""Paged key-value cache: attention over the rows that a search of the keys
finds, and eviction by attention weight.

A ``KvCache`` holds keys and values in pages of ``page_rows`` rows; a page table
(int32 [batch, columns]) names the pages of each sequence, ``lengths`` (int32
[batch]) its rows.  Rows are bf16, fp16, SQ8 (int8 codes with one f32 scale
max|x| * (1/127), symmetric by row like ``tessa.quantize_sq_int8_matrix``), or MX4
(4-bit floating point codes, two to a byte, with a power of two for each 32 dims).

* ``plan``           which pages a step's new rows go to and which come back; the
                     position, sequence and place (slot) of each token
* ``append``         new keys and values into the pages
* ``append_rotated`` the same by slot, with the norm of queries and keys for each head
                     and their rotation by position on the way
* ``read``           rows by slot, as values
* ``attend_prompt``  causal attention of the new tokens of each sequence, over all
                     rows or the first ``sinks`` and the last ``window``
* ``attend_token``   attention of one new token for each sequence; ``listed``
                     adds rows, e.g. those that ``graph.greedy_search`` found
                     among the keys; ``weights`` accumulates each row's attention
* ``evict``          keeps the first, the last and the most attended rows

Every computation happens in libtessa_hip.so, queued on the given or the current
stream; nothing waits for the device.  With ``stream`` the call's tensors are
marked as used there.  There are no gradients: tensors that require one are
refused while gradients are recorded.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import math
from dataclasses import dataclass, field
from typing import NamedTuple

import torch

from . import _native as N

_QUERY_TYPES = {torch.bfloat16: N.KV_BF16, torch.float16: N.KV_F16}
MX4 = torch.float4_e2m1fn_x2  # a cache's type: two 4-bit codes in each element
_SCALE = torch.float8_e8m0fnu  # of 32 dims of an MX4 row: a power of two
_TYPES = {torch.bfloat16: N.KV_BF16, torch.float16: N.KV_F16, torch.int8: N.KV_SQ8, MX4: N.KV_MX4}
_VALUE_TYPES = {**_QUERY_TYPES, torch.float32: N.KV_F32}
_INT = torch.int32
_MOST_ROWS = 2**30 - 1  # of a sequence, whatever its table covers


def _strides(t: torch.Tensor, count: int, each: int = 1):
    return (C.c_uint64 * count)(*(each * s for s in t.stride()[:count]))


@dataclass(frozen=True, eq=False)
class KvCache:
    """Pages of keys and values: [pages, heads, page_rows, head_dim] each, in
    any order of the first three dimensions (rows contiguous, 16-byte aligned);
    SQ8 caches carry f32 scales [pages, heads, page_rows].  MX4 caches have elements
    of two dims, [pages, heads, page_rows, head_dim / 2] (the even dim in the low bits; head_dim
    a multiple of 32), and carry float8_e8m0fnu scales [pages, heads, page_rows, head_dim / 32].
    A cache keeps the tensors that it was made of."""

    keys: torch.Tensor
    values: torch.Tensor
    key_scales: torch.Tensor | None = None
    value_scales: torch.Tensor | None = None
    _native: N.KvCache = field(init=False, repr=False)
    _scratch: dict = field(init=False, repr=False, default_factory=dict)  # bytes that calls of given sizes need

    def __post_init__(self):
        k, v = self.keys, self.values
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.dtype not in _TYPES:
            raise ValueError("keys and values must be bf16, fp16, int8 or float4_e2m1fn_x2 [pages, heads, page_rows, "
                             "head_dim], alike")
        if not k.is_cuda or k.device != v.device:
            raise ValueError("keys and values must be device tensors on one device")
        if k.stride(3) != 1 or v.stride(3) != 1:
            raise ValueError("rows must be contiguous")
        each = 2 if k.dtype == MX4 else 1  # dims of an element
        n = N.KvCache(type=_TYPES[k.dtype], pages=k.shape[0], heads=k.shape[1], page_rows=k.shape[2],
                      head_dim=each * k.shape[3], keys=k.data_ptr(), values=v.data_ptr(),
                      key_strides=_strides(k, 3, each), value_strides=_strides(v, 3, each))
        if k.dtype in (torch.int8, MX4):
            kind, name = (_SCALE, "MX4") if k.dtype == MX4 else (torch.float32, "SQ8")
            shape = (*k.shape[:3], n.head_dim // 32) if k.dtype == MX4 else k.shape[:3]
            for s in (self.key_scales, self.value_scales):
                if s is None or s.dtype != kind or s.shape != shape or s.device != k.device:
                    raise ValueError(f"an {name} cache needs {kind} scales [pages, heads, page_rows"
                                     + (", head_dim / 32]" if k.dtype == MX4 else "]"))
                if k.dtype == MX4 and shape[3] > 1 and s.stride(3) != 1:
                    raise ValueError("a row's scales must be contiguous")
            n.key_scales, n.value_scales = self.key_scales.data_ptr(), self.value_scales.data_ptr()
            n.key_scale_strides, n.value_scale_strides = _strides(self.key_scales, 3), _strides(self.value_scales, 3)
        elif self.key_scales is not None or self.value_scales is not None:
            raise ValueError("only SQ8 and MX4 caches have scales")
        object.__setattr__(self, "_native", n)

    @classmethod
    def allocate(cls, pages: int, heads: int, page_rows: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
                 device: str | torch.device = "cuda") -> "KvCache":
        if dtype == MX4 and head_dim % 32:
            raise ValueError(f"head_dim {head_dim} of an MX4 cache is not a multiple of 32")
        shape = (pages, heads, page_rows, head_dim // 2 if dtype == MX4 else head_dim)
        keys, values = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
        if dtype == MX4:
            return cls(keys, values, *(torch.empty((*shape[:3], head_dim // 32), dtype=_SCALE, device=device)
                                       for _ in range(2)))
        if dtype != torch.int8:
            return cls(keys, values)
        return cls(keys, values, *(torch.empty(shape[:3], dtype=torch.float32, device=device) for _ in range(2)))

    @property
    def page_rows(self) -> int:
        return int(self.keys.shape[2])

    @property
    def head_dim(self) -> int:
        return int(self._native.head_dim)

    @property
    def heads(self) -> int:
        return int(self.keys.shape[1])

    def _tensors(self):
        return self.keys, self.values, self.key_scales, self.value_scales


def _check(t: torch.Tensor, name: str, dtype: torch.dtype, shape: tuple, device) -> None:
    """A device tensor of the type and shape (None: any size), its last dimension contiguous."""
    got = t.shape
    alike = t.dtype is dtype and len(got) == len(shape)
    for w, g in zip(shape, got):
        alike = alike and (w is None or w == g)
    if not alike:
        want = ", ".join("*" if w is None else str(w) for w in shape)
        raise ValueError(f"{name} must be {dtype} [{want}], got {t.dtype} {list(got)}")
    if t.get_device() != device.index:
        raise ValueError(f"{name} must be on {device}, not {t.device}")
    if got[-1] > 1 and t.stride(-1) != 1 and t.numel():
        raise ValueError(f"the last dimension of {name} must be contiguous")


def _is(t: torch.Tensor, dtype: torch.dtype, shape: tuple, index: int) -> bool:
    """What ``_check`` asks for, as it mostly is: a small call's time is its checks'."""
    return t.dtype is dtype and t.shape == shape and t.get_device() == index and t.is_contiguous()


def _no_gradient(cache: KvCache, a: torch.Tensor, b: torch.Tensor | None = None) -> None:
    """There are no backward forms: a graph that would end here without a word is refused."""
    if (a.requires_grad or (b is not None and b.requires_grad) or cache.keys.requires_grad or cache.values.requires_grad
            or (cache.key_scales is not None and (cache.key_scales.requires_grad or cache.value_scales.requires_grad))):
        if torch.is_grad_enabled():
            raise ValueError("the key-value cache has no gradients: detach the tensors or call under torch.no_grad()")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t itself where its rows lie on 16-byte boundaries, else a copy of it."""
    s = t.stride()
    if s[2] == 1 and s[0] % 8 == 0 and s[1] % 8 == 0 and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _sequences(cache: KvCache, table: torch.Tensor, lengths: torch.Tensor, max_length: int | None) -> N.KvSequences:
    dev = cache.keys.device
    if not (table.dtype is _INT and table.dim() == 2 and table.get_device() == dev.index and table.is_contiguous()):
        _check(table, "page_table", _INT, (None, None), dev)
    batch, columns = table.shape
    if not (lengths.dtype is _INT and lengths.shape == (batch,) and lengths.get_device() == dev.index
            and lengths.is_contiguous()):
        _check(lengths, "lengths", _INT, (batch,), dev)
    covers = min(columns * cache._native.page_rows, _MOST_ROWS)
    if max_length is None:
        max_length = covers
    elif not 0 <= max_length <= covers:
        raise ValueError(f"max_length {max_length} is outside 0..{covers}, what the page table covers")
    return N.KvSequences(table.data_ptr(), lengths.data_ptr(), table.stride(0) if batch > 1 else columns, batch,
                         columns, max_length)


_HERE = contextlib.nullcontext()


def _on(stream: torch.cuda.Stream | None, device: torch.device, tensors):
    """The call's stream: (context in which it is current, its handle)."""
    if stream is None:
        handle = torch._C._cuda_getCurrentRawStream(device.index) or None
        return (_HERE if device.index == torch._C._cuda_getDevice() else torch.cuda.device(device)), handle
    if stream.device != device:
        raise ValueError(f"stream is on {stream.device}, the cache on {device}")
    for t in tensors:
        if t is not None:
            t.record_stream(stream)
    return torch.cuda.stream(stream), stream.cuda_stream or None


def _offsets(offsets: torch.Tensor, batch: int, device) -> None:
    _check(offsets, "offsets", torch.int32, (batch + 1,), device)


def append(cache: KvCache, page_table: torch.Tensor, starts: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
           offsets: torch.Tensor | None = None, max_new: int | None = None,
           stream: torch.cuda.Stream | None = None) -> None:
    """Rows ``starts[b]``.. of sequence b from tokens ``offsets[b]``..``offsets[b +
    1]`` of ``k`` and ``v`` ([tokens, heads, head_dim]); without ``offsets`` one token
    for each sequence.  ``max_new``: no sequence has more new tokens (default:
    all of them).  Rows past the page table are not written."""
    dev, native = cache.keys.device, cache._native
    _no_gradient(cache, k, v)
    seq = _sequences(cache, page_table, starts, None)
    dtype = cache.keys.dtype
    if dtype in (torch.int8, MX4):
        dtype = k.dtype if k.dtype in _QUERY_TYPES else torch.bfloat16
    tokens = k.shape[0] if k.dim() else 0
    shape = (tokens, native.heads, native.head_dim)
    for t, name in ((k, "k"), (v, "v")):
        if t.dtype != dtype or t.shape != shape or t.device != dev:
            raise ValueError(f"{name} must be {dtype} {list(shape)} on {dev}")
    if offsets is not None:
        _offsets(offsets, seq.batch, dev)
    elif tokens != seq.batch:
        raise ValueError(f"{tokens} tokens for {seq.batch} sequences without offsets")
    if max_new is None:
        max_new = tokens
    if max_new < 0:
        raise ValueError(f"max_new {max_new} is negative")
    on, handle = _on(stream, dev, (cache.keys, cache.values, cache.key_scales, cache.value_scales, page_table, starts, k, v,
                                   offsets))
    with on:
        k, v = _rows(k), _rows(v)
        new = N.KvTokens(k.data_ptr(), v.data_ptr(), k.stride()[:2], v.stride()[:2],
                         None if offsets is None else offsets.data_ptr(), tokens, min(max_new, tokens), _TYPES[dtype])
        N.check(N.load().tessa_kv_append(C.byref(cache._native), C.byref(seq), C.byref(new), handle), "kv append")


def _attend(cache, q, page_table, lengths, max_length, scale, sinks, window, stream, *, listed=None, weights=None,
            offsets=None, max_new=0, prompt=False):
    dev, lib, native = cache.keys.device, N.load(), cache._native
    _no_gradient(cache, q, weights)
    kind = _QUERY_TYPES.get(q.dtype)
    if q.dim() != 3 or kind is None or q.device != dev:
        raise ValueError(f"q must be bf16 or fp16 [tokens, q_heads, head_dim] on {dev}")
    if kind != native.type and native.type not in (N.KV_SQ8, N.KV_MX4):
        raise ValueError(f"q is {q.dtype}, the cache {cache.keys.dtype}")
    tokens, heads, dim = q.shape
    if dim != native.head_dim or heads == 0 or heads % native.heads:
        raise ValueError(f"q of {heads} heads x {dim} over a cache of {cache.heads} heads x {cache.head_dim}")
    if sinks < 0 or (window is not None and window < 0):
        raise ValueError(f"sinks {sinks} and window {window} must not be negative")
    seq = _sequences(cache, page_table, lengths, max_length)
    if prompt:
        _offsets(offsets, seq.batch, dev)
        max_new = tokens if max_new is None else max_new
        if max_new < 0:
            raise ValueError(f"max_new {max_new} is negative")
        max_new = min(max_new, tokens)
    elif tokens != seq.batch:
        raise ValueError(f"{tokens} queries for {seq.batch} sequences")
    if listed is not None:
        _check(listed, "listed", torch.int32, (seq.batch, cache.heads, None), dev)
        if window is None:
            raise ValueError("listed rows need a window: without one every row is visible")
        listed = listed if listed.shape[2] else None
    if weights is not None:
        _check(weights, "weights", torch.float32, (seq.batch, cache.heads, None), dev)
        if weights.shape[2] < seq.max_length:
            raise ValueError(f"weights of {weights.shape[2]} rows for lengths up to {seq.max_length}")
    on, handle = _on(stream, dev, (*cache._tensors(), q, page_table, lengths, listed, weights, offsets))
    with on:
        q = _rows(q)
        out = torch.empty(tokens, heads, dim, dtype=q.dtype, device=dev)
        lse = torch.empty(tokens, heads, dtype=torch.float32, device=dev)
        a = N.KvAttend(q.data_ptr(), out.data_ptr(), lse.data_ptr(), q.stride()[:2], (heads * dim, dim),
                       kind, heads, 1.0 / math.sqrt(dim) if scale is None else scale, min(sinks, seq.max_length),
                       N.KV_ALL if window is None else min(window, N.KV_ALL - 1), 0, None, None, (0, 0), None, tokens,
                       max_new, 0)
        if listed is not None:
            listed = listed.contiguous()
            a.listed, a.listed_count = listed.data_ptr(), listed.shape[2]
        if weights is not None:
            a.weights, a.weight_strides = weights.data_ptr(), weights.stride()[:2]
        if prompt:
            a.offsets = offsets.data_ptr()
        sizes = (prompt, seq.batch, seq.columns, seq.max_length, tokens, heads, max_new, a.sinks, a.window,
                 a.listed_count, weights is None)
        need = cache._scratch.get(sizes)
        if need is None:
            size = C.c_uint64(0)
            fn = lib.tessa_kv_attend_prompt_scratch if prompt else lib.tessa_kv_attend_token_scratch
            N.check(fn(C.byref(native), C.byref(seq), C.byref(a), C.byref(size)), "kv attend")
            if len(cache._scratch) >= 1024:
                cache._scratch.clear()
            need = cache._scratch[sizes] = size.value
        scratch = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        fn = lib.tessa_kv_attend_prompt if prompt else lib.tessa_kv_attend_token
        N.check(fn(C.byref(native), C.byref(seq), C.byref(a), scratch.data_ptr() if need else None, need, handle),
                "kv attend")
    return out, lse


def attend_token(q: torch.Tensor, cache: KvCache, page_table: torch.Tensor, lengths: torch.Tensor,
                 max_length: int | None = None, scale: float | None = None, sinks: int = 0, window: int | None = None,
                 listed: torch.Tensor | None = None, weights: torch.Tensor | None = None,
                 stream: torch.cuda.Stream | None = None):
    """(out [batch, q_heads, head_dim] in q's type, lse f32 [batch, q_heads]) of one
    query for each sequence, at its last row.  ``window`` None: all rows are
    visible; else the first ``sinks``, the last ``window`` and the rows that ``listed``
    (int32 [batch, heads, n], negative: none) names for each head of the cache,
    each once.  ``weights`` (f32 [batch, heads, >= max_length]) gets each row's
    weight added, summed over the head's queries.  ``max_length``: no sequence is
    longer (default: what the page table covers, at most 2^30 - 1); ``scale``
    1/sqrt(head_dim)."""
    return _attend(cache, q, page_table, lengths, max_length, scale, sinks, window, stream, listed=listed,
                   weights=weights)


def attend_prompt(q: torch.Tensor, offsets: torch.Tensor, cache: KvCache, page_table: torch.Tensor,
                  lengths: torch.Tensor, max_new: int | None = None, max_length: int | None = None,
                  scale: float | None = None, sinks: int = 0, window: int | None = None,
                  stream: torch.cuda.Stream | None = None):
    """(out [tokens, q_heads, head_dim] in q's type, lse f32 [tokens, q_heads]) of the
    new tokens of each sequence: tokens ``offsets[b]``..``offsets[b + 1]`` of q are
    its last rows, each seeing rows up to its own (with ``window``: the first
    ``sinks`` and its last ``window``).  Their keys and values are in the cache
    already; ``offsets`` cover all tokens (places past the last that they cover
    are not written).  ``max_new``: no sequence has more new tokens (default: all of them)."""
    return _attend(cache, q, page_table, lengths, max_length, scale, sinks, window, stream, offsets=offsets,
                   max_new=max_new, prompt=True)


def evict(cache: KvCache, page_table: torch.Tensor, lengths: torch.Tensor, weights: torch.Tensor, keep: int,
          sinks: int = 0, recent: int = 0, max_length: int | None = None, into: torch.Tensor | None = None,
          stream: torch.cuda.Stream | None = None):
    """(kept int32 [batch, heads, keep], lengths int32 [batch], weights f32 like
    ``weights``): of each head's rows of sequences longer than ``keep``, the first
    ``sinks``, the last ``recent`` and the most attended others move to rows 0.. in
    ascending order; ``kept`` names the rows they were (-1 past the new length), the
    new weights are theirs and zeros after them.  ``into``: the page table that they
    move to, its pages not among those read (default: in place; no page may then
    belong to two sequences).  Rows whose page id names no page do not stay, and
    rows that move to such an id are lost.  ``weights`` is left as it is."""
    dev = cache.keys.device
    _no_gradient(cache, weights)
    seq = _sequences(cache, page_table, lengths, max_length)
    _check(weights, "weights", torch.float32, (seq.batch, cache.heads, None), dev)
    rows = weights.shape[2]
    if keep <= 0 or sinks < 0 or recent < 0 or sinks + recent > keep:
        raise ValueError(f"keep {keep} must be positive and at least sinks {sinks} + recent {recent}")
    if rows < max(keep, seq.max_length):
        raise ValueError(f"weights of {rows} rows for lengths up to {seq.max_length}, keep {keep}")
    if into is not None:
        _check(into, "into", torch.int32, (seq.batch, None), dev)
        if into.shape[1] * cache.page_rows < min(keep, seq.max_length):
            raise ValueError(f"into covers {into.shape[1] * cache.page_rows} rows, {min(keep, seq.max_length)} stay")
    on, handle = _on(stream, dev, (*cache._tensors(), page_table, lengths, weights, into))
    with on:
        new_weights = torch.empty(seq.batch, cache.heads, rows, dtype=torch.float32, device=dev)
        kept = torch.empty(seq.batch, cache.heads, keep, dtype=torch.int32, device=dev)
        new_lengths = torch.empty(seq.batch, dtype=torch.int32, device=dev)
        e = N.KvEviction(weights.data_ptr(), weights.stride()[:2], new_weights.data_ptr(), kept.data_ptr(),
                         new_lengths.data_ptr(), None if into is None else into.data_ptr(),
                         0 if into is None else into.stride(0) if seq.batch > 1 else into.shape[1],
                         0 if into is None else into.shape[1], rows, keep, sinks, recent, 0)
        N.check(N.load().tessa_kv_evict(C.byref(cache._native), C.byref(seq), C.byref(e), handle), "kv evict")
    return kept, new_lengths, new_weights


def rotation_frequencies(dims: int, base: float = 10000.0, device: str | torch.device = "cuda") -> torch.Tensor:
    """f64 [dims / 2]: base^(-2i / dims) radians for each position, for ``append_rotated``."""
    return base ** (-torch.arange(0, dims, 2, dtype=torch.float64, device=device) / dims)


def append_rotated(cache: KvCache, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                   slots: torch.Tensor, frequencies: torch.Tensor | None = None, q_weight: torch.Tensor | None = None,
                   k_weight: torch.Tensor | None = None, eps: float = 1e-6, interleaved: bool = False,
                   stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """Queries, normalized and rotated, [tokens, q_heads, head_dim] in q's type; keys likewise, and values as they
    are, become the cache's rows ``slots`` (int64 [tokens]: page * page_rows + row, as ``plan`` gives them; others than
    the cache has are not written; no two tokens may have the same one).

    ``q_weight``, ``k_weight`` ([head_dim], q's type or f32): x * rsqrt(mean x^2 + eps) * weight
    for each head; None: no norm.  ``frequencies`` (f64 [r / 2], r a multiple of 16; None: no
    rotation): pair i of the first r dims turns by positions (int32 [tokens]) *
    frequencies[i] radians, dims (i, i + r / 2) or, ``interleaved``, (2i, 2i + 1).  All of it in f32
    (angles in 64 bits) and rounded once, so that the rows are what ``append`` makes of the rounded
    ones.  A token with a negative position is of no sequence: its queries come back as zeros and
    nothing of it is written."""
    dev, native = cache.keys.device, cache._native
    _no_gradient(cache, q, k)
    index, dtype = dev.index, q.dtype
    kind = _QUERY_TYPES.get(dtype)
    if q.dim() != 3 or kind is None or q.get_device() != index:
        raise ValueError(f"q must be bf16 or fp16 [tokens, q_heads, head_dim] on {dev}")
    if kind != native.type and native.type not in (N.KV_SQ8, N.KV_MX4):
        raise ValueError(f"q is {dtype}, the cache {cache.keys.dtype}")
    tokens, heads, dim = q.shape
    if dim != native.head_dim or heads == 0:
        raise ValueError(f"q of {heads} heads x {dim} for a cache of {cache.heads} heads x {cache.head_dim}")
    shape, each = (tokens, native.heads, dim), (tokens,)
    for t, name in ((k, "k"), (v, "v")):
        if t.dtype is not dtype or t.shape != shape or t.get_device() != index:
            raise ValueError(f"{name} must be {dtype} {list(shape)} on {dev}")
    if not (_is(positions, _INT, each, index) and _is(slots, torch.int64, each, index)):
        _check(positions, "positions", _INT, each, dev)
        _check(slots, "slots", torch.int64, each, dev)
    rotated, turns = 0, None
    if frequencies is not None:
        if not _is(frequencies, torch.float64, (frequencies.numel(),), index):
            _check(frequencies, "frequencies", torch.float64, (None,), dev)
        rotated, turns = 2 * frequencies.shape[0], frequencies.data_ptr()
        if rotated % 16 or rotated > dim:
            raise ValueError(f"{rotated} rotated dims must be a multiple of 16 up to {dim}")
    weight_type, weights = dtype, [0, 0]
    for i, w in enumerate((q_weight, k_weight)):
        if w is not None:
            weight_type = w.dtype if w.dtype is torch.float32 else dtype
            if not _is(w, weight_type, (dim,), index):
                _check(w, "k_weight" if i else "q_weight", weight_type, (dim,), dev)
            weights[i] = w.data_ptr()
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise ValueError(f"q_weight is {q_weight.dtype}, k_weight {k_weight.dtype}")
    for t in (v, frequencies, q_weight, k_weight):
        if t is not None and t.requires_grad:
            _no_gradient(cache, t)
    if not (eps >= 0.0 and math.isfinite(eps)):
        raise ValueError(f"eps {eps} must be finite and not negative")
    on, handle = _on(stream, dev, (*cache._tensors(), q, k, v, positions, slots, frequencies, q_weight, k_weight))
    with on:
        q, k, v = _rows(q), _rows(k), _rows(v)
        if weights[0] % 16 or weights[1] % 16:  # (clones start where an allocation does)
            own = [None if w is None else w.clone() for w in (q_weight, k_weight)]
            weights = [0 if w is None else w.data_ptr() for w in own]
        out = torch.empty(tokens, heads, dim, dtype=q.dtype, device=dev)
        a = N.KvRotated(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), q.stride()[:2], k.stride()[:2],
                        v.stride()[:2], (heads * dim, dim), positions.data_ptr(), slots.data_ptr(),
                        turns, weights[0] or None, weights[1] or None, tokens, kind, _VALUE_TYPES[weight_type],
                        heads, rotated, int(interleaved), eps)
        N.check(N.load().tessa_kv_append_rotated(C.byref(native), C.byref(a), handle), "kv append rotated")
    return out


def read(cache: KvCache, slots: torch.Tensor, dtype: torch.dtype | None = None, values: bool = True,
         stream: torch.cuda.Stream | None = None):
    """(keys, values) [n, heads, head_dim] of the cache's rows ``slots`` (int64 [n]: page * page_rows + row), zeros
    where the cache has no such row.  ``dtype``: bf16, fp16 or f32 (default: the cache's own, f32 for SQ8, bf16 for
    MX4, which holds each of its values).  ``values`` False: keys only, and None."""
    dev, native = cache.keys.device, cache._native
    _no_gradient(cache, slots)
    _check(slots, "slots", torch.int64, (None,), dev)
    if dtype is None:
        own = cache.keys.dtype
        dtype = torch.float32 if own == torch.int8 else torch.bfloat16 if own == MX4 else own
    if dtype not in _VALUE_TYPES:
        raise ValueError(f"rows are read as bf16, fp16 or f32, not {dtype}")
    on, handle = _on(stream, dev, (*cache._tensors(), slots))
    with on:
        shape = (slots.shape[0], native.heads, native.head_dim)
        k = torch.empty(shape, dtype=dtype, device=dev)
        v = torch.empty(shape, dtype=dtype, device=dev) if values else None
        a = N.KvRows(slots.data_ptr(), k.data_ptr(), v.data_ptr() if values else None, shape[0], _VALUE_TYPES[dtype], 0)
        N.check(N.load().tessa_kv_read(C.byref(native), C.byref(a), handle), "kv read")
    return k, v


class Plan(NamedTuple):
    """What a step does with its tokens (``plan``)."""

    lengths: torch.Tensor    # int32 [batch]: rows of each sequence after the step
    held: torch.Tensor       # int32 [batch]: pages of its table row that are its own
    count: torch.Tensor      # int32 [1]: free pages
    granted: torch.Tensor    # int32 [batch]: new rows that it got, all of them or none
    offsets: torch.Tensor    # int32 [batch + 1]: first token of each sequence
    positions: torch.Tensor  # int32 [tokens]: row of each token in its sequence, -1 where it got none
    sequences: torch.Tensor  # int32 [tokens], -1 past the last token
    slots: torch.Tensor      # int64 [tokens]: page * page_rows + row, -1 where the token got none


def plan(page_rows: int, page_table: torch.Tensor, lengths: torch.Tensor, held: torch.Tensor, new: torch.Tensor,
         free: torch.Tensor, count: torch.Tensor, tokens: int, stream: torch.cuda.Stream | None = None) -> Plan:
    """The pages and places of a step in which sequence b gets ``new[b]`` rows, or ends (negative).

    Sequence b has ``lengths[b]`` rows in the first ``held[b]`` pages of its row of ``page_table`` (int32 [batch,
    columns]); ``free`` (int32 [pages]) is a stack of ``count`` (int32 [1]) page ids that nobody holds.  ``tokens``:
    places of the step's tokens, which lie sequence by sequence; what is past the last is padding.

    In the order of the sequences, pages that one holds and needs no more (it ends, or was evicted from) go
    to the stack, then each that needs more gets them from its top, if what all up to it need is there.
    One that does not get its pages, or whose rows would pass the table's columns or tokens ``tokens``, is
    granted nothing: its tokens' places are -1 and its length stays (a prompt's attention of such tokens says
    nothing).  The table and the stack are changed in place, so they share no memory with each other or with other
    arguments; the lengths, held pages and count that go with them are the result's, and take the arguments' place in the
    next step."""
    dev = lengths.device
    if not lengths.is_cuda:
        raise ValueError("lengths must be a device tensor")
    if not 0 < page_rows <= 65536 or page_rows & (page_rows - 1):
        raise ValueError(f"page_rows must be a power of two in 1..65536, got {page_rows}")
    if not 0 <= tokens < 2**31:
        raise ValueError(f"tokens {tokens} is outside 0..2^31 - 1")
    i = dev.index
    if not (page_table.dim() == 2 and _is(page_table, _INT, page_table.shape, i)):
        _check(page_table, "page_table", _INT, (None, None), dev)
    batch, columns = page_table.shape
    each = (batch,)
    if not (_is(lengths, _INT, each, i) and _is(held, _INT, each, i) and _is(new, _INT, each, i)
            and _is(count, _INT, (1,), i)):
        for t, name, shape in ((lengths, "lengths", each), (held, "held", each), (new, "new", each),
                               (count, "count", (1,))):
            _check(t, name, _INT, shape, dev)
    if not _is(free, _INT, (free.numel(),), i):
        _check(free, "free", _INT, (None,), dev)
    on, handle = _on(stream, dev, (page_table, lengths, held, new, free, count))
    with on:
        slots = torch.empty(tokens, dtype=torch.int64, device=dev)
        sizes = [batch, batch, 1, batch, batch + 1, tokens, tokens]
        whole = torch.empty(4 * batch + 2 + 2 * tokens, dtype=_INT, device=dev)
        at, parts = whole.data_ptr(), whole.split_with_sizes(sizes)
        ints = (at, at + 4 * batch, at + 8 * batch, at + 8 * batch + 4, at + 12 * batch + 4, at + 16 * batch + 8,
                at + 16 * batch + 8 + 4 * tokens)
        a = N.KvStep(page_table.data_ptr(), page_table.stride(0) if batch > 1 else columns, lengths.data_ptr(),
                     held.data_ptr(), new.data_ptr(), free.data_ptr(), count.data_ptr(), *ints, slots.data_ptr(),
                     tokens, batch, columns, free.shape[0], page_rows)
        N.check(N.load().tessa_kv_plan(C.byref(a), handle), "kv plan")
    return Plan(*parts, slots)
