"""Eviction of sequences some of whose page ids name no page: such rows are not there,
before and after."""
import math

import numpy as np
import pytest
import torch

from gpu_helpers import require_gpu
from shear_amd import kvcache as KV
from test_gpu_kvcache import BF16, F16, SQ8, check_token, lens, normal, pool_with

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    return require_gpu()


def kept_rows(w, n, there, keep, sinks, recent):
    """The rows of one head that stay: those that are there, first and last before the heaviest."""
    rows = [j for j in range(n) if there[j]]
    if len(rows) <= keep:
        return rows
    always = [j for j in rows if j < sinks or j >= n - recent]
    middle = [j for j in rows if sinks <= j < n - recent]
    middle.sort(key=lambda j: (math.isnan(w[j]), 0.0 if math.isnan(w[j]) else -float(w[j]), j))
    return sorted(always + middle[: keep - len(always)])


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("cache_type,dim,page", [(BF16, 64, 16), (F16, 80, 8), (SQ8, 128, 16), (BF16, 256, 32)])
@pytest.mark.parametrize("keep,sinks,recent", [(100, 4, 30), (64, 32, 32), (1, 0, 1), (420, 20, 100), (900, 1, 500)])
def test_evict_with_missing_pages(gpu, in_place, cache_type, dim, page, keep, sinks, recent):
    lengths = [0, 60, 128, 500, 650, 899, 300]
    q_type = F16 if cache_type == F16 else BF16
    pool, g = pool_with(lengths, 2, page, dim, cache_type, q_type, keep + dim)
    rows, pages = 1000, pool.cache.keys.shape[0]
    # among the first rows, in the middle, among the last, all of a sequence
    pool.table_host[1, 0] = -1
    pool.table_host[2, 1] = pages
    pool.table_host[3, [0, 2, 499 // page]] = [2**30, -5, pages + 1]
    pool.table_host[4, [5, 6, 7]] = -1
    pool.table_host[5, 898 // page] = -(2**31)
    pool.table_host[6, :] = -1
    pool.table = torch.from_numpy(pool.table_host).cuda()
    w = np.exp(2 * g.standard_normal((len(lengths), 2, rows))).astype(np.float32)
    w[:, :, ::7] = 0.0
    w[:, :, 3::11] = 0.5  # ties
    w[4, 1, 10:600:3] = np.nan
    w[4, 0, 100:200] = -np.inf
    w[3, 0, 20:40] = np.inf  # (a part of them on a missing page)
    w[5, 1, :] = np.nan
    w[5, 0, :] = 0.0
    weights = torch.from_numpy(w).cuda()
    old = [[pool.rows(b, n, h) for h in range(2)] for b, n in enumerate(lengths)]
    into = None
    if not in_place:
        columns = -(-min(keep, 899) // page)
        extra = len(lengths) * columns
        cache = pool.cache  # a larger cache with the same pages first; what is not written is NaN (codes: scales)

        def grown(t):
            if t is None:
                return None
            more = torch.zeros((extra, *t.shape[1:]), dtype=t.dtype, device="cuda")
            return torch.cat([t, more if t.dtype == SQ8 else more.fill_(math.nan)])

        pool.cache = KV.KvCache(*(grown(t) for t in cache._tensors()))
        into_host = (pages + g.permutation(extra).reshape(len(lengths), columns)).astype(np.int32)
        into_host[4, 0] = -1  # its rows are lost
        into = torch.from_numpy(into_host).cuda()
        # ids that were past the last page would name new ones
        pool.table_host[pool.table_host >= pages] = -1
        pool.table = torch.from_numpy(pool.table_host).cuda()
    kept, new, moved = KV.evict(pool.cache, pool.table, lens(lengths), weights, keep, sinks=sinks, recent=recent,
                                max_length=899, into=into)
    kh, mh, nh = kept.cpu().numpy(), moved.cpu().numpy(), new.tolist()
    if into is not None:
        pool.table_host, pool.table = into_host, into
    for b, n in enumerate(lengths):
        for h in range(2):
            want = kept_rows(w[b, h], n, old[b][h][2], keep, sinks, recent)
            assert nh[b] == len(want)
            assert kh[b, h].tolist() == want + [-1] * (keep - len(want)), (b, h)
            assert np.array_equal(mh[b, h, : len(want)], w[b, h][want], equal_nan=True) and (mh[b, h, len(want):] == 0).all()
            k, v, there = pool.rows(b, len(want), h)
            assert np.array_equal(k[there], old[b][h][0][want][there]) and np.array_equal(v[there], old[b][h][1][want][there]), (b, h)
    # and what stays is what attention then sees
    q = normal(g, len(lengths), 4, dim, dtype=q_type)
    out, lse = KV.attend_token(q, pool.cache, pool.table, new)
    check_token(pool, nh, q, out, lse, None, 0)


@pytest.mark.parametrize("n,keep", [(40000, 9000), (33000, 200), (50000, 49000)])
def test_evict_long_with_missing_pages(gpu, n, keep):
    pool, g = pool_with([n], 2, 64, 16, BF16, BF16, n)
    pool.table_host[0, [0, 3, 77, 300, (n - 1) // 64]] = -1
    pool.table = torch.from_numpy(pool.table_host).cuda()
    old = [pool.rows(0, n, h) for h in range(2)]
    w = np.exp(2 * g.standard_normal((1, 2, n))).astype(np.float32)
    w[0, 1] = np.round(w[0, 1])
    kept, new, _ = KV.evict(pool.cache, pool.table, lens([n]), torch.from_numpy(w).cuda(), keep, sinks=70, recent=100,
                            max_length=n)
    for h in range(2):
        want = kept_rows(w[0, h], n, old[h][2], keep, 70, 100)
        assert new.tolist() == [len(want)] and kept[0, h].tolist() == want + [-1] * (keep - len(want))
        k, v, there = pool.rows(0, len(want), h)
        assert np.array_equal(k[there], old[h][0][want][there]) and np.array_equal(v[there], old[h][1][want][there])
