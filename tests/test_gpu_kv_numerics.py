"""The key-value cache's attention where weights, scales and values lie far apart: rows
that weigh little beside one that weighs much, SQ8 rows of very different size."""
import math

import numpy as np
import pytest
import torch

from gpu_helpers import require_gpu
from kv_reference import Pool
from shear_amd import kvcache as KV
from test_gpu_kvcache import BF16, F16, SQ8, check_prompt, check_token, lens, normal, prompt

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    return require_gpu()


def dominated(g, n, heads, dim, q_type, gap, at):
    """Keys and queries (two heads each): row ``at``'s logits lie ``gap`` above the others', which spread by about 1/4."""
    k = normal(g, n, heads, dim).float()
    q = normal(g, n, 2 * heads, dim).float() * 0.25
    k[..., 0], q[..., 0] = 0.0, 4.0
    k[at] = 0.0
    k[at, :, 0] = gap * math.sqrt(dim) / 4
    return q.to(q_type), k.to(q_type)


@pytest.mark.parametrize("q_type", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("size", [1.0, 0.05, 1e-3, "mixed"])
@pytest.mark.parametrize("gap", [0.0, 8.0])
def test_sq8_rows_beside_a_row_of_zeros(gpu, q_type, dim, size, gap):
    """A value row of zeros has scale 1, whatever the others' are; with a gap it takes most of the weight."""
    n = 700
    g = np.random.default_rng(dim)
    q, k = dominated(g, n, 1, dim, q_type, gap, 3)
    v = normal(g, n, 1, dim).float()
    v = v * (torch.from_numpy(10.0 ** g.uniform(-3, 1, (n, 1, 1))).float().cuda() if size == "mixed" else size)
    v[3] = 0.0
    pool = Pool(1, 11, 1, 64, dim, SQ8, 3)
    pool.fill([n], k, v.to(q_type))
    out, lse = prompt(pool, [n], [n], q)
    check_prompt(pool, [n], [n], q, out, lse, None, 0)
    out, lse = KV.attend_token(q[-1:].contiguous(), pool.cache, pool.table, lens([n]))
    check_token(pool, [n], q[-1:], out, lse, None, 0)
    weights = torch.zeros((1, 1, 704), device="cuda")  # (parts, and their join)
    out, lse = KV.attend_token(q[-1:].contiguous(), pool.cache, pool.table, lens([n]), weights=weights)
    check_token(pool, [n], q[-1:], out, lse, None, 0, gained=weights)


@pytest.mark.parametrize("q_type", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_sq8_value_row_that_is_nan_leaves_the_logits_alone(gpu, q_type, dim):
    n, bad = 400, (70, 200)
    g = np.random.default_rng(dim)
    k, v = normal(g, n, 1, dim, dtype=q_type), normal(g, n, 1, dim, dtype=q_type)
    q = normal(g, n, 2, dim, dtype=q_type)
    got = []
    for broken in (False, True):
        if broken:
            v[bad[0], 0, 5], v[bad[1], 0, 0] = math.inf, math.nan
        pool = Pool(1, 13, 1, 32, dim, SQ8, 4)
        pool.fill([n], k, v)
        weights = torch.zeros((2, 1, 416), device="cuda")
        two = pool.table.expand(2, -1).contiguous()
        out, lse = KV.attend_token(q[:2].contiguous(), pool.cache, two, lens([70, n]), weights=weights)
        got.append((*prompt(pool, [n], [n], q), *prompt(pool, [n], [n], q, window=60, sinks=2), out, lse, weights))
    clean, broken = got
    for i in (1, 3, 5, 6):
        assert torch.equal(clean[i], broken[i])
    rows = torch.arange(n, device="cuda")
    seen = rows >= bad[0]
    assert broken[0][seen].isnan().all() and torch.equal(broken[0][~seen], clean[0][~seen])
    seen = ((rows >= bad[0]) & (rows < bad[0] + 60)) | ((rows >= bad[1]) & (rows < bad[1] + 60))
    assert broken[2][seen].isnan().all() and torch.equal(broken[2][~seen], clean[2][~seen])
    assert torch.equal(broken[4][0], clean[4][0]) and broken[4][1].isnan().all()


@pytest.mark.parametrize("q_type", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("gap,size", [(12.0, 1.0), (16.0, 1.0), (18.0, 1.0), (22.0, 1.0), (16.0, 30.0)])
def test_rows_under_one_that_takes_the_weight(gpu, q_type, dim, gap, size):
    """A first row without a value takes almost all of the weight; the others' sum is the result."""
    n = 2000
    g = np.random.default_rng(dim)
    q, k = dominated(g, n, 1, dim, q_type, gap, 0)
    v = (normal(g, n, 1, dim).float() * size).to(q_type)
    v[0] = 0.0
    pool = Pool(1, 32, 1, 64, dim, q_type, 3)
    pool.fill([n], k, v)
    out, lse = prompt(pool, [n], [n], q)
    check_prompt(pool, [n], [n], q, out, lse, None, 0)


@pytest.mark.parametrize("q_type", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("gap,size", [(16.0, 1.0), (20.0, 30.0), (24.0, 30.0)])
@pytest.mark.parametrize("n", [500, 20000])
def test_token_rows_under_one_that_takes_the_weight(gpu, q_type, dim, gap, size, n):
    g = np.random.default_rng(dim)
    q, k = dominated(g, n, 1, dim, q_type, gap, n // 3)
    v = (normal(g, n, 1, dim).float() * size).to(q_type)
    v[n // 3] = 0.0
    pool = Pool(1, -(-n // 64), 1, 64, dim, q_type, 3)
    pool.fill([n], k, v)
    q = q[-1:].contiguous()
    weights = torch.zeros((1, 1, n), device="cuda")
    out, lse = KV.attend_token(q, pool.cache, pool.table, lens([n]), max_length=n, weights=weights)
    check_token(pool, [n], q, out, lse, None, 0, gained=weights)
    out, lse = KV.attend_token(q, pool.cache, pool.table, lens([n]), max_length=n)
    check_token(pool, [n], q, out, lse, None, 0)
