"""Attention over 4-bit rows whose logits are large: alike rows weigh alike, to the ends of f32, in every form of the kernels."""
import math

import numpy as np
import pytest
import torch

from gpu_helpers import require_gpu
from kv4_reference import Pool4
from kv_reference import ROUND
from shear_amd import kvcache as KV
from test_gpu_kvcache import BF16, F16, lens, normal

pytestmark = pytest.mark.gpu

# (queries' type, a key's value, a query's): a logit is the key as its codes hold it times the query, exactly.  2^127 is 2.5e38
# in base 2.
SIZES = [(BF16, 1e5, 1.0), (BF16, 1.6e6, 1.0), (BF16, 6.3e6, -1.0), (BF16, 3.1e7, 1.0), (BF16, 3.1e9, 1.0),
         (BF16, 6.4e9, -1.0), (BF16, 2.0**80, 1.0), (BF16, 2.0**127, 1.0), (BF16, 2.0**127, -1.0),
         (F16, 1.0, 60000.0), (F16, 600.0, 999.0), (F16, 50001.0, 99.0), (F16, 60000.0, 20000.0), (F16, 60000.0, -20000.0)]


@pytest.fixture(scope="module")
def gpu():
    return require_gpu()


def alike(n, page, q_type, size, seed):
    """n rows with keys of ``size`` in one dim, and their values (f64)."""
    dim = 64
    g = np.random.default_rng(seed)
    k = torch.zeros((n, 1, dim), dtype=torch.float64, device="cuda")
    k[..., 0] = size
    pool = Pool4(1, -(-n // page), 1, page, dim, 3)
    pool.fill([n], k, normal(g, n, 1, dim, dtype=q_type))
    keys, values, _ = pool.rows(0, n, 0)
    return pool, float(keys[0, 0]), torch.from_numpy(values).cuda()


# Weights are alike to the bit, as their logits are.  A chain of sums has less than 2^8 of them: 2^-16 of what is summed.
SUMS = 2.0**-16


@pytest.mark.parametrize("q_type,size,query", SIZES)
@pytest.mark.parametrize("group,page,window", [(1, 16, None), (4, 64, None), (8, 16, None), (20, 32, None), (3, 8, None),
                                               (16, 1, None), (4, 16, 100000)])
@pytest.mark.parametrize("n", [1, 130, 2001])
def test_tokens(gpu, q_type, size, query, group, page, window, n):
    pool, key, values = alike(n, page, q_type, size, 5)
    q = torch.zeros((1, group, 64), dtype=q_type, device="cuda")
    q[..., 0] = query
    logit, want = float(q[0, 0, 0]) * key, values.mean(0)
    weights = torch.zeros((1, 1, 2048), device="cuda")
    for kw in ({}, {"weights": weights}):
        out, lse = KV.attend_token(q, pool.cache, pool.table, lens([n]), scale=1.0, window=window, **kw)
        tol = ROUND[q_type] * want.abs() + SUMS * values.abs().mean(0) + (2.0**-25 if q_type == F16 else 0.0)
        assert ((out[0].double() - want).abs() <= 1.01 * tol).all()
        # the logit's rounding in base 2, that of its difference from the maximum, and the product with log(2): each half a unit
        assert ((lse.double() - logit - math.log(n)).abs() <= 2**-21 * abs(logit) + 2 * SUMS).all()
    w = weights[0, 0].double()
    # a group's weights of a row: numerator and sum alike, and as many additions as it has heads
    assert ((w[:n] - group / n).abs() <= 2 * SUMS * group / n).all() and (w[n:] == 0).all()


@pytest.mark.parametrize("q_type,size,query", SIZES)
@pytest.mark.parametrize("group,window", [(1, None), (2, None), (5, 4000)])
@pytest.mark.parametrize("n", [130, 700])
def test_prompts(gpu, q_type, size, query, group, window, n):
    pool, key, values = alike(n, 16, q_type, size, 6)
    q = torch.zeros((n, group, 64), dtype=q_type, device="cuda")
    q[..., 0] = query
    logit = float(q[0, 0, 0]) * key
    rows = torch.arange(1, n + 1, device="cuda").double()[:, None]
    want, spread = values.cumsum(0) / rows, values.abs().cumsum(0) / rows
    out, lse = KV.attend_prompt(q, lens([0, n]), pool.cache, pool.table, lens([n]), scale=1.0, window=window)
    u = ROUND[q_type]  # of the result, and of the weights
    tol = u * want.abs() + (u + SUMS) * spread + (2.0**-25 if q_type == F16 else 0.0)
    assert ((out.double() - want[:, None]).abs() <= 1.01 * tol[:, None]).all()
    assert ((lse.double() - logit - rows.log()).abs() <= 2**-21 * abs(logit) + 2 * SUMS).all()


@pytest.mark.parametrize("q_type,size,query", [s for s in SIZES if abs(s[1] * s[2]) < 1e10])
@pytest.mark.parametrize("group,page", [(2, 16), (7, 16), (17, 16), (2, 4)])
def test_tokens_beside_rows_that_weigh_nothing(gpu, q_type, size, query, group, page):
    """Half of the rows have a logit of zero or of the other sign: where the others' are positive these weigh nothing."""
    n = 400
    pool, key, values = alike(n, page, q_type, size, 7)
    kc = pool.bytes()[0]
    rows = np.arange(1, n, 2)
    at = torch.from_numpy(pool.table_host[0][rows // page].astype(np.int64)).cuda()
    kc[at, 0, torch.from_numpy(rows % page).cuda(), 0] ^= 8  # the sign of the first dim's code
    q = torch.zeros((1, group, 64), dtype=q_type, device="cuda")
    q[..., 0] = query
    logit = abs(float(q[0, 0, 0]) * key)
    seen = slice(0, n, 2) if query > 0 else slice(1, n, 2)
    want = values[seen].mean(0)
    weights = torch.zeros((1, 1, n), device="cuda")
    for kw in ({}, {"weights": weights}):
        out, lse = KV.attend_token(q, pool.cache, pool.table, lens([n]), scale=1.0, **kw)
        tol = ROUND[q_type] * want.abs() + SUMS * values.abs().mean(0) + (2.0**-25 if q_type == F16 else 0.0)
        assert ((out[0].double() - want).abs() <= 1.01 * tol).all()
        assert ((lse.double() - logit - math.log(n // 2)).abs() <= 2**-21 * logit + 2 * SUMS).all()
    w = weights[0, 0].double()
    assert ((w[seen] - 2 * group / n).abs() <= 2 * SUMS * 2 * group / n).all()
    assert abs(float(w.sum()) - group) <= 2 * SUMS * group
