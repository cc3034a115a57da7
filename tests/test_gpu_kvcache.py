"""The paged key-value cache on the GPU against 64-bit forms: append, attention
of single tokens and of prompts, eviction.  Unused slots of every cache hold NaN."""
import math

import numpy as np
import pytest
import torch

from gpu_helpers import require_gpu
from kv_reference import Pool, attend, close
from shear_amd import _native as N
from shear_amd import kvcache as KV
from shear_amd import tessa as T

pytestmark = pytest.mark.gpu

BF16, F16, SQ8 = torch.bfloat16, torch.float16, torch.int8


@pytest.fixture(scope="module")
def gpu():
    return require_gpu()


def normal(g, *shape, dtype=BF16, scale=1.0):
    return (torch.from_numpy(g.standard_normal(shape).astype(np.float32)) * scale).to(dtype).cuda()


def pool_with(lengths, heads, page, dim, cache_type, q_type, seed, columns=None, transposed=False):
    g = np.random.default_rng(seed)
    need = max(1, -(-max(lengths) // page))
    pool = Pool(len(lengths), columns or need, heads, page, dim, cache_type, seed, transposed=transposed)
    total = int(sum(lengths))
    if total:
        pool.fill(lengths, normal(g, total, heads, dim, dtype=q_type), normal(g, total, heads, dim, dtype=q_type))
    return pool, g


def lens(lengths):
    return torch.tensor(lengths, dtype=torch.int32, device="cuda")


def check_token(pool, lengths, q, out, lse, window, sinks, listed=None, gained=None):
    """Every (sequence, query head) against the 64-bit form; gained: what the weights grew by."""
    heads = pool.cache.heads
    group = q.shape[1] // heads
    dim = q.shape[2]
    qh, oh, lh = q.double().cpu().numpy(), out.double().cpu().numpy(), lse.double().cpu().numpy()
    for b, n in enumerate(lengths):
        for h in range(heads):
            k, v, there = pool.rows(b, n, h)
            j = np.arange(n)
            seen = np.ones(n, bool) if window is None else (j < sinks) | (j > n - 1 - window)
            if listed is not None:
                r = listed[b, h].cpu().numpy()
                seen[r[(r >= 0) & (r < n)]] = True
            seen &= there
            sums, worst = np.zeros(n), 0.0
            for i in range(h * group, (h + 1) * group):
                want, z, p, spread, delta = attend(qh[b, i], k, v, seen, 1 / math.sqrt(dim))
                assert close(oh[b, i], want, spread, delta, q.dtype, False).all(), (b, h, i, n)
                if z == -math.inf:
                    assert lh[b, i] == -math.inf, (b, h, i)
                else:
                    assert abs(lh[b, i] - z) <= delta + 2.0**-21 * (abs(z) + 1), (b, h, i)
                sums += p
                worst = max(worst, delta)
            if gained is not None:
                got = gained[b, h].double().cpu().numpy()
                assert (np.abs(got[:n] - sums) <= (2 * worst + 2.0**-19) * sums + 2.0**-23).all(), (b, h)
                assert (got[:n][~seen] == 0).all() and (got[n:] == 0).all()


@pytest.mark.parametrize("cache_type,q_type", [(BF16, BF16), (F16, F16), (SQ8, BF16), (SQ8, F16)])
@pytest.mark.parametrize("dim,group,heads,page", [
    (64, 1, 3, 16), (128, 8, 2, 64), (80, 3, 2, 1), (16, 17, 1, 32), (256, 4, 1, 128), (96, 40, 1, 16), (192, 2, 2, 8)])
def test_token_all_rows(gpu, cache_type, q_type, dim, group, heads, page):
    lengths = [0, 1, 2, 31, 32, 33, 127, 129, 700]
    pool, g = pool_with(lengths, heads, page, dim, cache_type, q_type, dim + group)
    q = normal(g, len(lengths), heads * group, dim, dtype=q_type, scale=2)
    out, lse = KV.attend_token(q, pool.cache, pool.table, lens(lengths))
    check_token(pool, lengths, q, out, lse, None, 0)


@pytest.mark.parametrize("cache_type,q_type", [(BF16, BF16), (SQ8, F16)])
@pytest.mark.parametrize("sinks,window", [(0, 1), (4, 100), (100, 0), (0, 0), (3, 5000), (64, 64)])
def test_token_window_list_and_weights(gpu, cache_type, q_type, sinks, window):
    lengths = [5, 0, 1000, 333, 64, 2500]
    pool, g = pool_with(lengths, 2, 32, 64, cache_type, q_type, 7 * sinks + window)
    q = normal(g, len(lengths), 6, 64, dtype=q_type, scale=2)
    rows = np.full((len(lengths), 2, 77), -1, np.int32)
    for b, n in enumerate(lengths):
        for h in range(2):
            some = g.permutation(max(n, 1) + 9)[:60]  # distinct, some past the length
            rows[b, h, g.permutation(77)[: len(some)]] = some
    listed = torch.from_numpy(rows).cuda()
    before = torch.rand((len(lengths), 2, 2560), device="cuda")
    weights = before.clone()
    out, lse = KV.attend_token(q, pool.cache, pool.table, lens(lengths), sinks=sinks, window=window, listed=listed,
                               weights=weights)
    zero = torch.zeros_like(weights)
    out0, lse0 = KV.attend_token(q, pool.cache, pool.table, lens(lengths), sinks=sinks, window=window, listed=listed,
                                 weights=zero)
    assert torch.equal(out, out0) and torch.equal(lse, lse0)
    assert torch.allclose(weights, before + zero, rtol=2**-22, atol=0)
    check_token(pool, lengths, q, out, lse, window, sinks, listed, zero)


@pytest.mark.parametrize("group", [1, 7, 20])
def test_token_weights_over_all_rows(gpu, group):
    # one sequence is split over many workgroups, the others end in the first
    lengths = [9000, 3, 0, 300]
    pool, g = pool_with(lengths, 2, 64, 128, BF16, BF16, group)
    q = normal(g, 4, 2 * group, 128, scale=2)
    weights = torch.zeros((4, 2, 9024), device="cuda")
    out, lse = KV.attend_token(q, pool.cache, pool.table, lens(lengths), weights=weights)
    check_token(pool, lengths, q, out, lse, None, 0, None, weights)


def test_token_pages_that_are_none_and_lengths_out_of_range(gpu):
    lengths = [300, 300, 300]
    pool, g = pool_with(lengths, 2, 16, 64, BF16, BF16, 3)
    pages = pool.cache.keys.shape[0]
    pool.table_host[0, 3:5] = -1
    pool.table_host[1, :] = pages  # past the last
    pool.table_host[2, 18] = 2**30
    pool.table = torch.from_numpy(pool.table_host).cuda()
    q = normal(g, 3, 4, 64)
    weights = torch.zeros((3, 2, 304), device="cuda")
    out, lse = KV.attend_token(q, pool.cache, pool.table, lens(lengths), weights=weights)
    check_token(pool, lengths, q, out, lse, None, 0, None, weights)
    assert (out[1] == 0).all() and (lse[1] == -math.inf).all()
    # negative: none; longer than max_length: clipped to it
    out, lse = KV.attend_token(q, pool.cache, pool.table, lens([-5, 2**31 - 1, 2**31 - 1]), max_length=290)
    assert (out[0] == 0).all() and (lse[0] == -math.inf).all()
    check_token(pool, [0, 290, 290], q, out, lse, None, 0)


@pytest.mark.parametrize("q_type,cache_type", [(BF16, BF16), (F16, SQ8)])
def test_token_values_that_are_not_finite(gpu, q_type, cache_type):
    """A row that is NaN reaches its own sequence and head only; logits of -inf weigh nothing."""
    lengths = [200, 200]
    pool, g = pool_with(lengths, 2, 16, 64, cache_type, q_type, 5)
    k = normal(g, 1, 2, 64, dtype=q_type)
    v = normal(g, 1, 2, 64, dtype=q_type)
    v[0, 1, 3] = float("nan")
    KV.append(pool.cache, pool.table[:1], lens([150]), k, v)
    q = normal(g, 2, 4, 64, dtype=q_type)
    out, lse = KV.attend_token(q, pool.cache, pool.table, lens(lengths))
    assert out[0, 2:].isnan().any() and not out[0, :2].isnan().any() and not out[1].isnan().any()
    # outside of the window it does nothing
    out, lse = KV.attend_token(q, pool.cache, pool.table, lens(lengths), sinks=100, window=49)
    check_token(pool, lengths, q, out, lse, 49, 100)
    if cache_type != SQ8:
        # logits of -inf: key of -inf against queries that are positive there
        k = torch.zeros_like(k)
        k[..., 0] = -math.inf
        KV.append(pool.cache, pool.table[1:], lens([20]), k, normal(g, 1, 2, 64, dtype=q_type))
        q = q.abs() + 0.01
        out, lse = KV.attend_token(q, pool.cache, pool.table, lens(lengths))
        # (the rest of the -inf row's products are 0: the logit is -inf)
        assert not out[1].isnan().any()
        check_one = [pool.rows(1, 200, h) for h in range(2)]
        for i in range(4):
            kk, vv, _ = check_one[i // 2]
            want, z, _, spread, delta = attend(q[1, i].double().cpu().numpy(), kk, vv, np.arange(200) != 20, 0.125)
            assert close(out[1, i].double().cpu().numpy(), want, spread, delta, q_type, False).all()
        # a sequence of that row alone is one that sees nothing
        out, lse = KV.attend_token(q[1:], pool.cache, pool.table[1:], lens([21]), window=1)
        assert (out == 0).all() and (lse == -math.inf).all()


def test_token_large_logits_and_scales_far_apart(gpu):
    """Logits of +-2,000 and SQ8 scales over 20 orders of magnitude."""
    g = np.random.default_rng(11)
    n = 500
    for cache_type, q_type in ((BF16, BF16), (SQ8, BF16)):
        pool = Pool(1, 8, 2, 64, 64, cache_type, 1)
        size = torch.from_numpy(10.0 ** g.uniform(-10, 10, (n, 2, 1))).float().cuda()
        k, v = normal(g, n, 2, 64, scale=30), (normal(g, n, 2, 64).float() * size).to(q_type)
        pool.fill([n], k, v)
        q = normal(g, 1, 4, 64, scale=30)
        out, lse = KV.attend_token(q, pool.cache, pool.table, lens([n]))
        check_token(pool, [n], q, out, lse, None, 0)
        # small logits, so that every row counts
        q = normal(g, 1, 4, 64, scale=0.001)
        out, lse = KV.attend_token(q, pool.cache, pool.table, lens([n]))
        check_token(pool, [n], q, out, lse, None, 0)


def test_token_strides_and_scale(gpu):
    """Row-major pages, queries as views of larger tensors (aligned or not), a page table with a stride, a scale."""
    lengths = [70, 400]
    pool, g = pool_with(lengths, 3, 16, 64, BF16, BF16, 21, transposed=True)
    assert pool.cache.keys.stride(2) > pool.cache.keys.stride(1)
    wide = torch.full((2, pool.table.shape[1] + 5), -7, dtype=torch.int32, device="cuda")
    wide[:, : pool.table.shape[1]] = pool.table
    table = wide[:, : pool.table.shape[1]]
    q = normal(g, 2, 9, 64)
    want = KV.attend_token(q, pool.cache, pool.table, lens(lengths))
    check_token(pool, lengths, q, *want, None, 0)
    big = torch.zeros((2, 2, 9, 72), dtype=BF16, device="cuda")
    big[:, 1, :, 3:67] = q
    big2 = torch.zeros((9, 2, 80), dtype=BF16, device="cuda")
    big2[:, :, 8:72] = q.transpose(0, 1)
    for view in (big[:, 1, :, 3:67], big2.transpose(0, 1)[:, :, 8:72]):
        got = KV.attend_token(view, pool.cache, table, lens(lengths))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    half = KV.attend_token(q, pool.cache, pool.table, lens(lengths), scale=0.0625)
    doubled = KV.attend_token(q * 0.5, pool.cache, pool.table, lens(lengths))
    assert torch.equal(half[0], doubled[0]) and torch.equal(half[1], doubled[1])


def test_token_and_append_past_32_bits(gpu):
    """Pages whose places pass 2^32 bytes and 2^31 elements."""
    pages = 5 * 2**30 // (2 * 128 * 128 * 2)
    keys = torch.empty((pages, 2, 128, 128), dtype=BF16, device="cuda")
    values = torch.empty_like(keys)
    assert keys.numel() > 2**31
    cache = KV.KvCache(keys, values)
    ids = [pages - 1, 3, pages - 2, pages // 2 + 1]
    table = torch.tensor([ids], dtype=torch.int32, device="cuda")
    g = np.random.default_rng(2)
    n = 450
    k, v = normal(g, n, 2, 128), normal(g, n, 2, 128)
    KV.append(cache, table, lens([0]), k, v, offsets=lens([0, n]))
    assert torch.equal(keys[pages - 1, :, :, :].transpose(0, 1), k[:128])
    assert torch.equal(values[pages // 2 + 1, :, : n - 384].transpose(0, 1), v[384:])
    q = normal(g, 1, 4, 128)
    out, lse = KV.attend_token(q, cache, table, lens([n]))
    small = Pool(1, 4, 2, 128, 128, BF16, 0)
    small.fill([n], k, v)
    want = KV.attend_token(q, small.cache, small.table, lens([n]))
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    off = lens([0, n])
    got, _ = KV.attend_prompt(k.repeat_interleave(2, 1), off, cache, table, lens([n]))
    want, _ = KV.attend_prompt(k.repeat_interleave(2, 1), off, small.cache, small.table, lens([n]))
    assert torch.equal(got, want)


def test_stream_and_graph(gpu):
    """On a stream of its own, and captured in a graph that is replayed between eager work."""
    lengths = [900, 100]
    pool, g = pool_with(lengths, 2, 32, 128, BF16, BF16, 31)
    q = normal(g, 2, 8, 128)
    n = lens(lengths)
    want, want_lse = KV.attend_token(q, pool.cache, pool.table, n, weights=torch.zeros((2, 2, 928), device="cuda"))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got, lse = KV.attend_token(q, pool.cache, pool.table, n, stream=side)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(lse, want_lse)
    weights = torch.zeros((2, 2, 928), device="cuda")
    k, v = normal(g, 2, 2, 128), normal(g, 2, 2, 128)
    off = lens([0, 40, 50])
    pq = normal(g, 50, 8, 128)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        KV.append(pool.cache, pool.table, n - 1, k, v)
        out, lse = KV.attend_token(q, pool.cache, pool.table, n, weights=weights)
        prompt, _ = KV.attend_prompt(pq, off, pool.cache, pool.table, n, max_new=40)
        kept, new, moved = KV.evict(pool.cache, pool.table, n, weights, 64, sinks=2, recent=8)
    for rep in range(3):
        weights.zero_()
        fill_k, fill_v = normal(np.random.default_rng(rep), 1000, 2, 128), normal(np.random.default_rng(rep + 9), 1000, 2, 128)
        pool.fill(lengths, fill_k, fill_v)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (out, lse, weights, prompt, kept, new, moved)]
        pool.fill(lengths, fill_k, fill_v)
        KV.append(pool.cache, pool.table, n - 1, k, v)
        w = torch.zeros_like(weights)
        eager = [*KV.attend_token(q, pool.cache, pool.table, n, weights=w), w]
        eager.append(KV.attend_prompt(pq, off, pool.cache, pool.table, n, max_new=40)[0])
        eager += KV.evict(pool.cache, pool.table, n, w, 64, sinks=2, recent=8)
        torch.cuda.synchronize()
        for a, b in zip(got, eager):
            assert torch.equal(a, b), rep


def check_prompt(pool, lengths, new, q, out, lse, window, sinks):
    heads = pool.cache.heads
    group, dim = q.shape[1] // heads, q.shape[2]
    qh, oh, lh = q.double().cpu().numpy(), out.double().cpu().numpy(), lse.double().cpu().numpy()
    t0 = 0
    for b, (n, fresh) in enumerate(zip(lengths, new)):
        for h in range(heads):
            k, v, there = pool.rows(b, n, h)
            j = np.arange(n)
            picks = range(fresh) if fresh <= 64 else sorted({0, 1, 2, fresh // 3, fresh // 2, fresh - 2, fresh - 1,
                                                              *range(29, fresh, max(1, fresh // 23))})
            for i in picks:
                pos = n - fresh + i
                seen = (j <= pos) & there
                if window is not None:
                    seen &= (j < sinks) | (j > pos - window)
                for a in range(h * group, (h + 1) * group):
                    want, z, _, spread, delta = attend(qh[t0 + i, a], k, v, seen, 1 / math.sqrt(dim))
                    ok = close(oh[t0 + i, a], want, spread, delta, q.dtype, True)
                    assert ok.all(), (b, h, i, a, pos)
                    if z == -math.inf:
                        assert lh[t0 + i, a] == -math.inf, (b, h, i)
                    else:
                        assert abs(lh[t0 + i, a] - z) <= delta + 2.0**-21 * (abs(z) + 1), (b, h, i)
        t0 += fresh


def prompt(pool, lengths, new, q, **kw):
    off = lens(np.concatenate([[0], np.cumsum(new)]).tolist())
    return KV.attend_prompt(q, off, pool.cache, pool.table, lens(lengths), **kw)


@pytest.mark.parametrize("cache_type,q_type", [(BF16, BF16), (F16, F16), (SQ8, BF16), (SQ8, F16)])
@pytest.mark.parametrize("dim,group,heads,page", [
    (64, 1, 2, 16), (128, 4, 2, 64), (80, 3, 1, 8), (16, 7, 1, 32), (256, 2, 1, 128), (192, 1, 2, 1)])
def test_prompt_causal(gpu, cache_type, q_type, dim, group, heads, page):
    new = [1, 0, 33, 200, 64, 5]
    lengths = [1, 40, 33, 263, 300, 700]
    pool, g = pool_with(lengths, heads, page, dim, cache_type, q_type, dim + group)
    q = normal(g, sum(new), heads * group, dim, dtype=q_type, scale=2)
    out, lse = prompt(pool, lengths, new, q, max_new=200)
    check_prompt(pool, lengths, new, q, out, lse, None, 0)


@pytest.mark.parametrize("cache_type,q_type", [(BF16, BF16), (SQ8, F16)])
@pytest.mark.parametrize("sinks,window", [(0, 1), (4, 100), (70, 0), (0, 0), (0, 64), (200, 65), (5, 100000)])
def test_prompt_window_and_sinks(gpu, cache_type, q_type, sinks, window):
    new, lengths = [300, 20, 128], [300, 1000, 129]
    pool, g = pool_with(lengths, 2, 32, 64, cache_type, q_type, sinks + window)
    q = normal(g, sum(new), 6, 64, dtype=q_type, scale=2)
    out, lse = prompt(pool, lengths, new, q, sinks=sinks, window=window)
    check_prompt(pool, lengths, new, q, out, lse, window, sinks)


@pytest.mark.parametrize("cache_type", [BF16, SQ8])
@pytest.mark.parametrize("window,sinks", [(None, 0), (3000, 10)])
def test_prompt_few_tokens_over_a_long_cache(gpu, cache_type, window, sinks):
    # split over the rows and joined
    new, lengths = [6, 1], [9000, 2500]
    pool, g = pool_with(lengths, 2, 64, 128, cache_type, BF16, 17)
    q = normal(g, 7, 8, 128, scale=2)
    out, lse = prompt(pool, lengths, new, q, sinks=sinks, window=window)
    check_prompt(pool, lengths, new, q, out, lse, window, sinks)


@pytest.mark.parametrize("q_type,cache_type", [(BF16, BF16), (F16, SQ8)])
@pytest.mark.parametrize("dim", [16, 64, 80, 128, 144, 256])
@pytest.mark.parametrize("window,sinks", [(None, 0), (700, 5)])
def test_prompt_many_queries_over_a_longer_cache(gpu, q_type, cache_type, dim, window, sinks):
    # split over the rows, and 1,760 queries to join
    new, lengths = [150, 70], [1100, 900]
    pool, g = pool_with(lengths, 2, 32, dim, cache_type, q_type, dim)
    q = normal(g, 220, 8, dim, dtype=q_type, scale=2)
    out, lse = prompt(pool, lengths, new, q, max_new=150, sinks=sinks, window=window)
    check_prompt(pool, lengths, new, q, out, lse, window, sinks)


@pytest.mark.parametrize("columns,rows", [(60, 512), (60, 513), (72, 576), (72, 577), (256, 2048), (256, 2049)])
def test_token_on_both_sides_of_whole_columns(gpu, columns, rows):
    g = np.random.default_rng(columns)
    lengths = [rows, 0, 1, rows - 1] + g.integers(0, 90, columns // 4 - 4).tolist()
    pool, g = pool_with(lengths, 4, 64, 32, BF16, BF16, rows)
    q = normal(g, columns // 4, 8, 32, scale=2)
    out, lse = KV.attend_token(q, pool.cache, pool.table, lens(lengths), max_length=rows)
    check_token(pool, lengths, q, out, lse, None, 0)


def test_prompt_more_tokens_than_rows_and_missing_pages(gpu):
    new, lengths = [10, 150, 40], [4, 150, 40]
    pool, g = pool_with(lengths, 1, 16, 64, BF16, BF16, 23)
    pool.table_host[1, 2:4] = -1
    pool.table_host[2, 0] = 2**30
    pool.table = torch.from_numpy(pool.table_host).cuda()
    q = normal(g, 200, 2, 64)
    out, lse = prompt(pool, lengths, new, q)
    check_prompt(pool, lengths, new, q, out, lse, None, 0)
    assert (out[:6] == 0).all() and (lse[:6] == -math.inf).all()  # tokens before row 0 see nothing


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q_type,cache_type", [(BF16, BF16), (F16, F16), (BF16, SQ8)])
def test_prompt_values_that_only_later_queries_see(gpu, dim, q_type, cache_type):
    """Infinities and NaN reach the queries that see their row, and no other."""
    n = 150
    g = np.random.default_rng(dim)
    pool = Pool(1, 10, 1, 16, dim, cache_type, 4)
    k, v = normal(g, n, 1, dim, dtype=q_type), normal(g, n, 1, dim, dtype=q_type)
    v[70, 0, 5], v[70, 0, dim - 1] = math.inf, -math.inf
    v[90, 0, 7] = math.nan
    k[120, 0, 2] = math.nan
    pool.fill([n], k, v)
    q = normal(g, n, 2, dim, dtype=q_type)
    out, lse = prompt(pool, [n], [n], q)
    if cache_type == SQ8:  # a row with such a value is NaN altogether
        assert not out[:70].isnan().any() and out[70:].isnan().all()
        return
    check_prompt(pool, [70], [70], q[:70], out[:70], lse[:70], None, 0)
    assert (out[70:90, :, 5] == math.inf).all() and (out[70:90, :, dim - 1] == -math.inf).all()
    keep = [d for d in range(dim) if d not in (5, 7, dim - 1)]
    clean = Pool(1, 10, 1, 16, dim, cache_type, 4)
    v2 = v.clone()
    v2[70, 0, 5] = v2[70, 0, dim - 1] = v2[90, 0, 7] = 0
    clean.fill([n], k, v2)
    want, want_lse = prompt(clean, [n], [n], q)
    assert torch.equal(out[:120, :, keep], want[:120, :, keep]) and torch.equal(lse[:120], want_lse[:120])
    assert out[90:, :, 7].isnan().all() and not out[:90].isnan().any()
    assert out[120:].isnan().all() and lse[120:].isnan().all()
    # a window that has left them behind
    out, lse = prompt(pool, [n], [n], q, window=10)
    assert not out[80:90].isnan().any() and not out[100:120].isnan().any() and not out[130:].isnan().any()
    assert torch.isfinite(out[80:90]).all() and torch.isfinite(out[130:]).all()


@pytest.mark.parametrize("cache_type", [BF16, SQ8])
@pytest.mark.parametrize("dim,page", [(128, 64), (128, 16), (64, 32), (256, 128), (64, 128)])
def test_prompt_missing_pages_of_every_size(gpu, cache_type, dim, page):
    # a tile in one page, of several pages, and smaller than one
    new, lengths = [200, 40, 3], [700, 650, 500]
    pool, g = pool_with(lengths, 2, page, dim, cache_type, BF16, dim + page)
    pool.table_host[0, 1] = -1
    pool.table_host[0, 4] = 2**30
    pool.table_host[1, 0] = -(2**31)
    pool.table_host[2, :] = -1
    pool.table = torch.from_numpy(pool.table_host).cuda()
    q = normal(g, sum(new), 4, dim, scale=2)
    out, lse = prompt(pool, lengths, new, q)
    check_prompt(pool, lengths, new, q, out, lse, None, 0)
    assert (out[240:] == 0).all() and (lse[240:] == -math.inf).all()
    out, lse = prompt(pool, lengths, new, q, sinks=3, window=90)
    check_prompt(pool, lengths, new, q, out, lse, 90, 3)


@pytest.mark.parametrize("dim,page", [(64, 128), (128, 64), (256, 32)])
@pytest.mark.parametrize("q_type", [BF16, F16])
def test_prompt_values_not_finite_in_pages_of_whole_tiles(gpu, dim, page, q_type):
    """As above where a tile lies in one page: a column with such a value is infinite or NaN
    from the query on that sees the row, and the others are the results without it."""
    n = 400
    g = np.random.default_rng(dim + page)
    k, v = normal(g, n, 1, dim, dtype=q_type), normal(g, n, 1, dim, dtype=q_type)
    q = normal(g, n, 2, dim, dtype=q_type)
    plain = Pool(1, 16, 1, page, dim, q_type, 6)
    plain.fill([n], k, v)
    want, want_lse = prompt(plain, [n], [n], q)
    check_prompt(plain, [n], [n], q, want, want_lse, None, 0)
    v[75, 0, 0], v[140, 0, dim - 1], v[300, 0, 9] = math.inf, -math.inf, math.nan
    pool = Pool(1, 16, 1, page, dim, q_type, 6)
    pool.fill([n], k, v)
    out, lse = prompt(pool, [n], [n], q)
    rest = [d for d in range(dim) if d not in (0, 9, dim - 1)]
    assert torch.equal(out[:, :, rest], want[:, :, rest]) and torch.equal(lse, want_lse)
    for row, col, of in ((75, 0, torch.isposinf), (140, dim - 1, torch.isneginf), (300, 9, torch.isnan)):
        assert torch.equal(out[:row, :, col], want[:row, :, col]) and of(out[row:, :, col]).all(), (row, col)


@pytest.mark.parametrize("cache_type,q_type", [(BF16, BF16), (F16, F16), (SQ8, BF16), (SQ8, F16)])
@pytest.mark.parametrize("dim,page", [(128, 64), (64, 16)])
@pytest.mark.parametrize("how", ["grow", "fall", "jump", "low"])
def test_prompt_maxima_that_move(gpu, cache_type, q_type, dim, page, how):
    """Logits that grow along the rows, that fall, that jump by hundreds within a
    tile, and that are all far below zero."""
    n, new = 640, 640
    g = np.random.default_rng(dim)
    j = np.arange(n)
    size = {"grow": j / 40, "fall": (n - j) / 40, "jump": np.where(j % 200 == 170, 60.0, 1.0), "low": np.ones(n)}[how]
    q = normal(g, new, 2, dim, dtype=q_type)
    k = normal(g, n, 1, dim)
    if how in ("jump", "low"):  # keys along the queries' common part
        q[:, :, 0], k[:, :, 0] = 4, (-100 if how == "low" else 4)
    k = (k.float() * torch.from_numpy(size.astype(np.float32)).cuda()[:, None, None]).to(q_type)
    v = normal(g, n, 1, dim, dtype=q_type)
    pool = Pool(1, -(-n // page), 1, page, dim, cache_type, 9)
    pool.fill([n], k, v)
    out, lse = prompt(pool, [n], [new], q)
    check_prompt(pool, [n], [new], q, out, lse, None, 0)
    out, lse = KV.attend_token(q[-1:].contiguous(), pool.cache, pool.table, lens([n]))
    check_token(pool, [n], q[-1:], out, lse, None, 0)


@pytest.mark.parametrize("window,sinks", [(None, 0), (200, 2)])
def test_token_many_sequences(gpu, window, sinks):
    # more sequences than a workgroup has threads, most of them short, some empty
    g = np.random.default_rng(3)
    lengths = g.integers(0, 60, 700).tolist()
    lengths[5], lengths[300], lengths[699] = 1500, 900, 513
    pool, g = pool_with(lengths, 1, 64, 32, BF16, BF16, 12)
    q = normal(g, 700, 3, 32, scale=2)
    weights = torch.zeros((700, 1, 1600), device="cuda")
    out, lse = KV.attend_token(q, pool.cache, pool.table, lens(lengths), sinks=sinks, window=window, weights=weights)
    check_token(pool, lengths, q, out, lse, window, sinks, gained=weights)
    bare, bare_lse = KV.attend_token(q, pool.cache, pool.table, lens(lengths), sinks=sinks, window=window)
    check_token(pool, lengths, q, bare, bare_lse, window, sinks)


def test_prompt_agrees_with_single_tokens(gpu):
    lengths = [257, 64]
    pool, g = pool_with(lengths, 2, 32, 128, BF16, BF16, 41)
    q = normal(g, 2, 8, 128)
    a, la = prompt(pool, lengths, [1, 1], q)
    b, lb = KV.attend_token(q, pool.cache, pool.table, lens(lengths))
    check_prompt(pool, lengths, [1, 1], q, a, la, None, 0)
    check_token(pool, lengths, q, b, lb, None, 0)


def sq8_rule(x):
    """Codes and scales of rows: f32 product and quotient, rounded half away from zero."""
    x = x.float().cpu().numpy()
    top = np.abs(x).max(-1)
    scale = np.where(top > 0, top * (np.float32(1) / np.float32(127)), np.float32(1)).astype(np.float32)
    q = (x / scale[:, None]).astype(np.float32)
    return (np.sign(q) * np.floor(np.abs(q).astype(np.float64) + 0.5)).astype(np.int8), scale


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [16, 80, 128, 240])
def test_append(gpu, dtype, dim):
    """Ragged tokens land in their rows and nowhere else; SQ8 rows follow the rule bit for
    bit, and the set quantizer's within the last place of the scale."""
    g = np.random.default_rng(dim)
    new, start = [5, 0, 40, 1], [0, 3, 17, 63]
    k, v = normal(g, 46, 3, dim, dtype=dtype), normal(g, 46, 3, dim, dtype=dtype)
    k[3, 1] = 0  # a row of zeros
    k[7, 2, 1::2] = k[7, 2, 0] / 2  # ties of the rounding
    off = lens(np.concatenate([[0], np.cumsum(new)]).tolist())
    for cache_type in (dtype, SQ8):
        pool = Pool(4, 4, 3, 16, dim, cache_type, 1)
        KV.append(pool.cache, pool.table, lens(start), k, v, offsets=off, max_new=40)
        written = torch.zeros(pool.cache.keys.shape[:3], dtype=torch.bool, device="cuda")
        t = 0
        for b, (n, s) in enumerate(zip(new, start)):
            for i in range(n):
                page, slot = int(pool.table_host[b, (s + i) // 16]), (s + i) % 16
                written[page, :, slot] = True
                for x, y, sc in ((pool.cache.keys, k, pool.cache.key_scales), (pool.cache.values, v, pool.cache.value_scales)):
                    if cache_type != SQ8:
                        assert torch.equal(x[page, :, slot], y[t])
                    else:
                        codes, scales = sq8_rule(y[t])
                        assert np.array_equal(x[page, :, slot].cpu().numpy(), codes)
                        assert np.array_equal(sc[page, :, slot].cpu().numpy(), scales)
                        near = T.quantize_sq_int8_matrix(y[t].float())
                        assert int((x[page, :, slot].int() - near.codes[:, :dim].int()).abs().max()) <= 1
                        assert torch.allclose(sc[page, :, slot], near.scales, rtol=2**-23, atol=0)
                t += 1
        rest = pool.cache.key_scales if cache_type == SQ8 else pool.cache.keys.float().sum(-1)
        assert rest[~written].isnan().all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("mixed", [False, True])
def test_append_codes_of_every_magnitude(gpu, dtype, mixed):
    """The rule bit for bit: maxima of every significand and of exponents over the type's
    range, subnormal ones among them, alone or next to others in a wave."""
    g = np.random.default_rng(8)
    n, heads, dim = 4096, 2, 64
    x = torch.from_numpy(g.integers(0, 65536, (n, heads, dim)).astype(np.uint16).view(np.int16)).view(dtype).float()
    x = torch.where(torch.isfinite(x), x, torch.zeros(()))
    low, high = (-133, 126) if dtype == BF16 else (-24, 14)
    size = g.integers(low, high, (n, heads, 1)) if mixed else np.repeat(np.sort(g.integers(low, high, (n, 1, 1)), 0), 2, 1)
    # significands in 1..2, at most eight powers of two below the row's maximum
    frac = torch.frexp(x)[0].double() * 2 * torch.from_numpy(2.0 ** -g.integers(0, 9, (n, heads, dim)))
    k = (frac * torch.from_numpy(2.0 ** size.astype(np.float64))).to(dtype)
    assert torch.isfinite(k).all()
    pool = Pool(1, n // 64, heads, 64, dim, SQ8, 2)
    k = k.cuda()
    pool.fill([n], k, -k)
    y = k.float().cpu().numpy()
    top = np.abs(y).max(-1)
    scale = (top * (np.float32(1) / np.float32(127))).astype(np.float32)
    scale = np.where(scale > 0, scale, np.float32(1))
    q = (y / scale[..., None]).astype(np.float32).astype(np.float64)
    codes = np.clip(np.sign(q) * np.floor(np.abs(q) + 0.5), -127, 127)
    page, slot = pool.table_host[0, np.arange(n) // 64].astype(np.int64), np.arange(n) % 64
    for rows, scales, sign in ((pool.cache.keys, pool.cache.key_scales, 1), (pool.cache.values, pool.cache.value_scales, -1)):
        assert (scales.cpu().numpy()[page, :, slot] == scale).all()
        assert (rows.cpu().numpy()[page, :, slot] == sign * codes).all()


def test_append_single_tokens_rows_past_the_table_and_not_finite(gpu):
    g = np.random.default_rng(3)
    pool = Pool(3, 2, 2, 8, 32, BF16, 2)
    before = pool.cache.keys.clone()
    k, v = normal(g, 3, 2, 32), normal(g, 3, 2, 32)
    KV.append(pool.cache, pool.table, lens([15, 16, -1]), k, v)  # the last two lie outside
    assert torch.equal(pool.cache.keys[int(pool.table_host[0, 1]), :, 7], k[0])
    same = pool.cache.keys.view(torch.int16) == before.view(torch.int16)
    assert int((~same).any(-1).sum()) == 2  # one slot, two heads
    sq8 = Pool(1, 1, 2, 8, 32, SQ8, 2)
    k[0, 0, 4], v[0, 1, 0] = math.inf, math.nan
    KV.append(sq8.cache, sq8.table, lens([2]), k[:1], v[:1])
    page = int(sq8.table_host[0, 0])
    assert sq8.cache.key_scales[page, :, 2].isnan().tolist() == [True, False]
    assert sq8.cache.value_scales[page, :, 2].isnan().tolist() == [False, True]
    assert (sq8.cache.keys[page, 0, 2] == 0).all()


def kept_rows(w, n, keep, sinks, recent):
    """The rows of one head that stay, by a stable sort in 64 bits."""
    if n <= keep:
        return list(range(n))
    middle = range(sinks, n - recent)
    key = [(-math.inf if math.isnan(w[j]) else float(w[j])) for j in middle]
    nan = [math.isnan(w[j]) for j in middle]
    best = sorted(range(len(key)), key=lambda i: (nan[i], -key[i] if not nan[i] else 0.0, i))[: keep - sinks - recent]
    return sorted([*range(sinks), *(middle[i] for i in best), *range(n - recent, n)])


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("cache_type,dim,page", [(BF16, 64, 16), (F16, 80, 8), (SQ8, 128, 64), (BF16, 256, 1)])
@pytest.mark.parametrize("keep,sinks,recent", [(100, 4, 30), (100, 0, 0), (64, 32, 32), (1, 0, 0), (1, 0, 1), (900, 1, 500)])
def test_evict(gpu, in_place, cache_type, dim, page, keep, sinks, recent):
    lengths = [0, 1, 100, 101, 650, 899]
    q_type = F16 if cache_type == F16 else BF16
    pool, g = pool_with(lengths, 2, page, dim, cache_type, q_type, keep + dim)
    rows = 1000
    w = np.exp(2 * g.standard_normal((len(lengths), 2, rows))).astype(np.float32)
    w[:, :, ::7] = 0.0
    w[:, :, 3::11] = 0.5  # ties
    w[4, 1, 10:600:3] = np.nan
    w[4, 0, 100:200] = -0.0
    w[5, 0, 50] = np.inf
    w[5, 1, :] = 1.0
    weights = torch.from_numpy(w).cuda()
    old = [[pool.rows(b, n, h) for h in range(2)] for b, n in enumerate(lengths)]
    into = None
    if not in_place:
        columns = -(-min(keep, 899) // page)
        extra = len(lengths) * columns
        cache = pool.cache  # a larger cache with the same pages first
        def grown(t):
            if t is None:
                return None
            return torch.cat([t, torch.zeros((extra, *t.shape[1:]), dtype=t.dtype, device="cuda")])
        first = cache.keys.shape[0]
        pool.cache = KV.KvCache(*(grown(t) for t in cache._tensors()))
        into_host = first + g.permutation(extra).reshape(len(lengths), columns).astype(np.int32)
        into = torch.from_numpy(into_host.astype(np.int32)).cuda()
    kept, new, moved = KV.evict(pool.cache, pool.table, lens(lengths), weights, keep, sinks=sinks, recent=recent,
                                max_length=899, into=into)
    assert torch.equal(weights.view(torch.int32), torch.from_numpy(w).cuda().view(torch.int32))
    assert new.tolist() == [min(n, keep) for n in lengths]
    kh, mh = kept.cpu().numpy(), moved.cpu().numpy()
    if into is not None:
        pool.table_host, pool.table = into_host, into
    for b, n in enumerate(lengths):
        for h in range(2):
            want = kept_rows(w[b, h], n, keep, sinks, recent)
            assert kh[b, h].tolist() == want + [-1] * (keep - len(want)), (b, h)
            assert np.array_equal(mh[b, h, : len(want)], w[b, h][want], equal_nan=True) and (mh[b, h, len(want):] == 0).all()
            got = pool.rows(b, len(want), h)
            assert np.array_equal(got[0], old[b][h][0][want]) and np.array_equal(got[1], old[b][h][1][want]), (b, h)


@pytest.mark.parametrize("in_place", [False, True])
def test_evict_over_tables_of_more_rows_than_32_bits_count(gpu, in_place):
    # 65,536 columns of 65,536 rows, of which the sequence uses the first
    g = np.random.default_rng(2)
    cache = KV.KvCache.allocate(2, 1, 65536, 16)
    table, into = (torch.full((1, 65536), -1, dtype=torch.int32, device="cuda") for _ in range(2))
    table[0, 0], into[0, 0] = 0, 1
    k, v = normal(g, 900, 1, 16), normal(g, 900, 1, 16)
    KV.append(cache, table, lens([0]), k, v, offsets=lens([0, 900]))
    w = torch.from_numpy(g.random((1, 1, 1000)).astype(np.float32)).cuda()
    kept, n, _ = KV.evict(cache, table, lens([900]), w, 300, sinks=2, recent=10, max_length=900,
                          into=None if in_place else into)
    want = kept_rows(w[0, 0].cpu().numpy(), 900, 300, 2, 10)
    out, lse = KV.attend_token(k[:1].contiguous(), cache, table, lens([1]), window=4)  # (with the default max_length)
    assert torch.equal(out, cache.values[0, :, :1].transpose(0, 1))
    assert n.tolist() == [300] and kept[0, 0].tolist() == want
    page = 0 if in_place else 1
    assert torch.equal(cache.keys[page, 0, :300], k[kept[0, 0].long(), 0])
    assert torch.equal(cache.values[page, 0, :300], v[kept[0, 0].long(), 0])


@pytest.mark.parametrize("n,keep", [(32768 + 40, 9000), (40000, 39999), (100001, 20000), (33000, 200)])
def test_evict_long(gpu, n, keep):
    """Around and above the number of candidates held in registers; in place over many steps."""
    g = np.random.default_rng(n)
    pool = Pool(1, -(-n // 64), 2, 64, 16, BF16, 1, spare=0)
    k, v = normal(g, n, 2, 16), normal(g, n, 2, 16)
    pool.fill([n], k, v)
    w = np.exp(2 * g.standard_normal((1, 2, n))).astype(np.float32)
    w[0, 1] = np.round(w[0, 1])  # many ties
    kept, new, moved = KV.evict(pool.cache, pool.table, lens([n]), torch.from_numpy(w).cuda(), keep, sinks=4, recent=33,
                                max_length=n)
    for h in range(2):
        middle = w[0, h, 4: n - 33].astype(np.float64)
        order = np.argsort(-middle, kind="stable")[: keep - 37]
        want = np.concatenate([np.arange(4), np.sort(order) + 4, np.arange(n - 33, n)])
        assert np.array_equal(kept[0, h].cpu().numpy(), want)
        at = torch.from_numpy(want).cuda()
        got = pool.rows(0, keep, h)
        assert np.array_equal(got[0], k[at, h].double().cpu().numpy())
        assert np.array_equal(got[1], v[at, h].double().cpu().numpy())


def test_refusals(gpu):
    pool, g = pool_with([40, 20], 2, 16, 64, BF16, BF16, 1)
    c, t, n = pool.cache, pool.table, lens([40, 20])
    q = normal(g, 2, 4, 64)
    k = normal(g, 2, 2, 64)
    bad = [
        lambda: KV.attend_token(q.half(), c, t, n),
        lambda: KV.attend_token(q.float(), c, t, n),
        lambda: KV.attend_token(q[:, :3], c, t, n),
        lambda: KV.attend_token(q[:1], c, t, n),
        lambda: KV.attend_token(q[:, :, :32], c, t, n),
        lambda: KV.attend_token(q.cpu(), c, t, n),
        lambda: KV.attend_token(q, c, t.long(), n),
        lambda: KV.attend_token(q, c, t, n.long()),
        lambda: KV.attend_token(q, c, t, n[:1]),
        lambda: KV.attend_token(q, c, t, n, max_length=10_000),
        lambda: KV.attend_token(q, c, t, n, window=-1),
        lambda: KV.attend_token(q, c, t, n, sinks=-1, window=3),
        lambda: KV.attend_token(q, c, t, n, listed=torch.zeros((2, 2, 3), dtype=torch.int32, device="cuda")),
        lambda: KV.attend_token(q, c, t, n, window=3, listed=torch.zeros((2, 1, 3), dtype=torch.int32, device="cuda")),
        lambda: KV.attend_token(q, c, t, n, weights=torch.zeros((2, 2, 47), device="cuda")),
        lambda: KV.attend_token(q, c, t, n, weights=torch.zeros((2, 2, 48), device="cuda", dtype=BF16)),
        lambda: KV.attend_prompt(q, lens([0, 2]), c, t, n),
        lambda: KV.attend_prompt(q, lens([0, 1, 2]).long(), c, t, n),
        lambda: KV.attend_prompt(q, lens([0, 1, 2]), c, t, n, max_new=-1),
        lambda: KV.append(c, t, n, k.half(), k.half()),
        lambda: KV.append(c, t, n, k[:1], k[:1]),
        lambda: KV.append(c, t, n, k, k[:, :1]),
        lambda: KV.evict(c, t, n, torch.zeros((2, 2, 48), device="cuda"), 0),
        lambda: KV.evict(c, t, n, torch.zeros((2, 2, 48), device="cuda"), 8, sinks=5, recent=4),
        lambda: KV.evict(c, t, n, torch.zeros((2, 2, 40), device="cuda"), 8),
        lambda: KV.evict(c, t, n, torch.zeros((2, 2, 48), device="cuda"), 20, into=t[:, :1]),
        lambda: KV.KvCache(c.keys, c.values.half()),
        lambda: KV.KvCache(c.keys, c.values, c.keys.float()[..., 0], c.keys.float()[..., 0]),
        lambda: KV.KvCache(c.keys.to(torch.int8), c.values.to(torch.int8)),
        lambda: KV.KvCache(c.keys.transpose(2, 3), c.values.transpose(2, 3)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    odd = KV.KvCache.allocate(4, 2, 16, 72)  # a head dimension that the kernels do not have
    with pytest.raises(RuntimeError, match="head_dim"):
        KV.attend_token(torch.zeros((2, 2, 72), dtype=BF16, device="cuda"), odd, t, n)
    odd = KV.KvCache.allocate(4, 2, 12, 64)
    with pytest.raises(RuntimeError, match="page_rows"):
        KV.attend_token(q, odd, t, n)
    with pytest.raises(RuntimeError, match="scale"):
        KV.attend_token(q, c, t, n, scale=0.0)
    # nothing to do is no error
    none = torch.zeros((0, 3), dtype=torch.int32, device="cuda")
    out, lse = KV.attend_token(q[:0], c, none, n[:0])
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    KV.append(c, none, n[:0], k[:0], k[:0])
    out, lse = KV.attend_prompt(q[:0], lens([0, 0, 0]), c, t, n)
    assert out.shape == (0, 4, 64)
    kept, new, _ = KV.evict(c, none, n[:0], torch.zeros((0, 2, 48), device="cuda"), 8)
    assert kept.shape == (0, 2, 8) and new.shape == (0,)


def test_a_cache_keeps_its_tensors(gpu):
    pool, g = pool_with([20], 2, 16, 64, BF16, BF16, 1)
    for name in ("keys", "values", "key_scales"):
        with pytest.raises(AttributeError):
            setattr(pool.cache, name, torch.zeros_like(pool.cache.keys))
    q = normal(g, 1, 4, 64)
    shared = torch.zeros((1, 1, 32), device="cuda").expand(1, 2, 32)  # one sum for both heads
    with pytest.raises(N.TessaError, match="weight strides"):
        KV.attend_token(q, pool.cache, pool.table, lens([20]), weights=shared)
