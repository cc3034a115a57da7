"""The key-value cache's attention where weights, scales and values lie far apart: rows
that weigh little beside one that weighs much, SQ8 rows of very different size."""
import math

import numpy as np
import pytest
import torch

from gpu_helpers import require_gpu
from kv_reference import Pool
from shear_amd import kvcache as KV
from test_gpu_kvcache import BF16, F16, SQ8, check_prompt, check_token, lens, normal, pool_with, prompt

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


def with_values(v, rows):
    """Copy of v [n, 1, dim] whose values (row, dim) -> x of ``rows`` are x, and the columns that have any."""
    v = v.clone()
    for (row, d), x in rows.items():
        v[row, 0, d] = x
    return v, sorted({d for _, d in rows})


def settled(rows, seen, d):
    """What the values of column d that are not finite make of a sum over the rows that ``seen`` marks, 0: nothing."""
    return sum((x for (row, col), x in rows.items() if col == d and seen[row]), 0.0)


def check_special(out, clean, rows, seen):
    """One query: columns are infinite or NaN as the seen values make them, and else as without them."""
    for d in range(out.shape[-1]):
        want = settled(rows, seen, d)
        if want == 0.0:
            assert (out[..., d] == clean[..., d]).all(), d
        elif math.isnan(want):
            assert out[..., d].isnan().all(), d
        else:
            assert (out[..., d] == want).all(), d


@pytest.mark.parametrize("q_type", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 80, 128, 256])
@pytest.mark.parametrize("n,gap", [(500, 0.0), (500, 40.0), (500, 80.0), (9000, 0.0), (9000, 40.0)])
def test_token_values_that_are_infinite(gpu, q_type, dim, n, gap):
    """An infinity reaches the result as it is, however small its row's weight, and NaN or both signs as NaN."""
    g = np.random.default_rng(dim)
    q, k = dominated(g, n, 1, dim, q_type, gap, n - 30)
    rows = {(5, 0): math.inf, (n - 1, 1): -math.inf, (n // 2, dim - 1): math.nan, (9, 7): math.inf, (n - 2, 7): math.inf,
            (n - 30, 20): -math.inf, (11, 33): math.inf, (n - 40, 33): -math.inf, (200, 50): -math.inf}
    plain = normal(g, n, 1, dim, dtype=q_type)
    v, cols = with_values(plain, rows)
    plain[:, :, cols] = torch.where(torch.isfinite(v[:, :, cols]), plain[:, :, cols], 0)
    q = q[-1:].contiguous()
    listed = torch.tensor([[[5, 200, 17]]], dtype=torch.int32, device="cuda")
    got = []
    for values in (plain, v):
        pool = Pool(1, -(-n // 64), 1, 64, dim, q_type, 3)
        pool.fill([n], k, values)
        weights = torch.zeros((1, 1, n), device="cuda")
        got.append((KV.attend_token(q, pool.cache, pool.table, lens([n]), max_length=n),
                    KV.attend_token(q, pool.cache, pool.table, lens([n]), max_length=n, weights=weights),
                    KV.attend_token(q, pool.cache, pool.table, lens([n]), max_length=n, window=60, sinks=4, listed=listed)))
    j = np.arange(n)
    near = (j < 4) | (j >= n - 60) | (j == 5) | (j == 200) | (j == 17)
    for i, seen in ((0, j >= 0), (1, j >= 0), (2, near)):
        assert torch.equal(got[0][i][1], got[1][i][1])
        check_special(got[1][i][0], got[0][i][0], rows, seen)


@pytest.mark.parametrize("q_type", [BF16, F16])
@pytest.mark.parametrize("dim,page", [(64, 16), (80, 64), (128, 64), (256, 32)])
@pytest.mark.parametrize("n,new,gap", [(400, 400, 0.0), (400, 400, 40.0), (400, 400, 80.0), (5000, 3, 0.0), (5000, 3, 40.0),
                                       (900, 300, 40.0)])
def test_prompt_values_that_are_infinite(gpu, q_type, dim, page, n, new, gap):
    g = np.random.default_rng(dim)
    q, k = dominated(g, n, 1, dim, q_type, gap, 60)
    rows = {(5, 0): math.inf, (n - 1, 1): -math.inf, (n // 2, dim - 1): math.nan, (9, 7): math.inf, (n - 2, 7): math.inf,
            (60, 20): -math.inf, (11, 33): math.inf, (n - 40, 33): -math.inf, (200, 50): -math.inf}
    plain = normal(g, n, 1, dim, dtype=q_type)
    v, cols = with_values(plain, rows)
    plain[:, :, cols] = torch.where(torch.isfinite(v[:, :, cols]), plain[:, :, cols], 0)
    q = q[n - new:].contiguous()
    got = []
    for values in (plain, v):
        pool = Pool(1, -(-n // page), 1, page, dim, q_type, 3)
        pool.fill([n], k, values)
        got.append((prompt(pool, [n], [new], q), prompt(pool, [n], [new], q, window=150, sinks=7)))
    j = np.arange(n)
    for i, window in ((0, None), (1, 150)):
        (out, lse), (clean, clean_lse) = got[1][i], got[0][i]
        assert torch.equal(lse, clean_lse)
        for t in sorted({0, 1, 2, new - 1, new - 2, new // 2, *range(3, new, max(1, new // 40))} & set(range(new))):
            pos = n - new + t
            seen = (j <= pos) if window is None else (j <= pos) & ((j < 7) | (j > pos - window))
            check_special(out[t].cpu(), clean[t].cpu(), rows, seen)


@pytest.mark.parametrize("cache_type,q_type", [(BF16, BF16), (F16, F16), (SQ8, BF16), (SQ8, F16)])
@pytest.mark.parametrize("dim", [144, 256])
@pytest.mark.parametrize("group", [14, 16, 17, 40])
def test_token_whole_blocks_of_heads_of_wide_rows(gpu, cache_type, q_type, dim, group):
    """16 heads of 256 dims take more LDS than a kernel has by default; whole columns and shared rows."""
    lengths = [300, 1, 0, 129]
    pool, g = pool_with(lengths, 2, 16, dim, cache_type, q_type, dim + group)
    q = normal(g, len(lengths), 2 * group, dim, dtype=q_type, scale=2)
    out, lse = KV.attend_token(q, pool.cache, pool.table, lens(lengths))
    check_token(pool, lengths, q, out, lse, None, 0)
    weights = torch.zeros((len(lengths), 2, 304), device="cuda")
    out, lse = KV.attend_token(q, pool.cache, pool.table, lens(lengths), weights=weights)
    check_token(pool, lengths, q, out, lse, None, 0, gained=weights)


@pytest.mark.parametrize("cache_type,q_type,size,sign", [
    (BF16, BF16, 2.2e38, -1.0), (SQ8, BF16, 2.2e38, -1.0), (BF16, BF16, 2.2e38, 1.0), (BF16, BF16, 3.1e7, 1.0),
    (F16, F16, 60000.0, -20000.0), (F16, F16, 60000.0, 20000.0), (F16, F16, 50001.0, 99.0), (SQ8, F16, 60000.0, 20000.0)])
def test_logits_of_any_size(gpu, cache_type, q_type, size, sign):
    """Rows whose logits are alike weigh as much as each other, to the ends of f32 (2.2e38 is 3.2e38 in base 2)."""
    n, dim = 130, 64
    g = np.random.default_rng(5)
    k = torch.zeros((n, 1, dim), dtype=q_type, device="cuda")
    k[..., 0] = size
    q = torch.zeros((n, 2, dim), dtype=q_type, device="cuda")
    q[..., 0] = sign
    v = normal(g, n, 1, dim, dtype=q_type)
    pool = Pool(1, 3, 1, 64, dim, cache_type, 3)
    pool.fill([n], k, v)
    values = torch.from_numpy(pool.rows(0, n, 0)[1]).cuda()
    want = values.cumsum(0) / torch.arange(1, n + 1, device="cuda")[:, None]
    out, lse = KV.attend_prompt(q, lens([0, n]), pool.cache, pool.table, lens([n]), scale=1.0)
    logit = float(q[0, 0, 0]) * pool.rows(0, 1, 0)[0][0, 0]
    # a rounding of the result and one of the weights, which are all alike
    assert ((out[:, 0].double() - want).abs() <= 2**-8 * want.abs() + (2**-8 + 2**-19) * values.abs().mean() + 1e-6).all()
    rows = torch.arange(1, n + 1, device="cuda").double()[:, None]
    assert ((lse.double() - logit - rows.log()).abs() <= 2**-21 * abs(logit)).all()
    weights = torch.zeros((1, 1, 192), device="cuda")
    for kw in ({}, {"weights": weights}):
        out, lse = KV.attend_token(q[:1], pool.cache, pool.table, lens([n]), scale=1.0, **kw)
        assert ((out[0].double() - want[-1]).abs() <= 2**-8 * want[-1].abs() + 2**-17).all()
        assert ((lse.double() - logit - math.log(n)).abs() <= 2**-21 * abs(logit)).all()
    assert torch.allclose(weights[0, 0, :n], torch.full((n,), 2.0 / n, device="cuda"), rtol=2**-20, atol=0)


@pytest.mark.parametrize("group", [3, 4])
def test_weights_of_rows_without_a_page_beside_nan(gpu, group):
    """A key that is NaN makes the weights NaN, but not those of rows that are not there or not seen."""
    n = 300
    pool, g = pool_with([n], 1, 16, 64, BF16, BF16, group)
    k = normal(g, 1, 1, 64)
    k[0, 0, 3] = math.nan
    KV.append(pool.cache, pool.table, lens([150]), k, k)
    pool.table_host[0, 4:6] = -1
    pool.table = torch.from_numpy(pool.table_host).cuda()
    q = normal(g, 1, group, 64)
    weights = torch.ones((1, 1, 304), device="cuda")
    out, _ = KV.attend_token(q, pool.cache, pool.table, lens([n]), weights=weights)
    w = weights[0, 0]
    assert out.isnan().all() and (w[64:96] == 1).all() and (w[n:] == 1).all()
    assert w[:64].isnan().all() and w[96:n].isnan().all()
    weights.fill_(1)
    KV.attend_token(q, pool.cache, pool.table, lens([n]), window=200, sinks=70, weights=weights)
    assert (w[64:100] == 1).all() and w[:64].isnan().all() and w[100:n].isnan().all()


@pytest.mark.parametrize("cache_type", [BF16, SQ8])
@pytest.mark.parametrize("size", [3e38, 1e-22])
@pytest.mark.parametrize("how", ["level", "grow", "same"])
def test_values_near_the_ends_of_bf16(gpu, cache_type, size, how):
    """Values as large as bf16 has them stay finite sums while the maximum of the logits moves; small ones keep their bits."""
    n, dim = 640, 64
    g = np.random.default_rng(7)
    q, k = normal(g, n, 2, dim), normal(g, n, 1, dim)
    if how == "grow":
        k = (k.float() * torch.linspace(0, 12, n, device="cuda")[:, None, None]).bfloat16()
    v = (torch.from_numpy(g.uniform(0.5, 1.0, (n, 1, dim)).astype(np.float32)).cuda() * size).bfloat16()
    if how != "same":
        v = v * torch.from_numpy(g.choice([-1.0, 1.0], (n, 1, dim))).cuda().bfloat16()
    pool = Pool(1, 10, 1, 64, dim, cache_type, 3)
    pool.fill([n], k, v)
    out, lse = prompt(pool, [n], [n], q)
    check_prompt(pool, [n], [n], q, out, lse, None, 0)
    for kw in ({}, {"weights": torch.zeros((1, 1, n), device="cuda")}):
        out, lse = KV.attend_token(q[-1:].contiguous(), pool.cache, pool.table, lens([n]), **kw)
        check_token(pool, [n], q[-1:], out, lse, None, 0)


@pytest.mark.parametrize("cache_type,q_type", [(BF16, BF16), (F16, F16), (SQ8, BF16), (SQ8, F16)])
@pytest.mark.parametrize("n", [2, 6])
def test_token_sums_that_cancel(gpu, cache_type, q_type, n):
    """Many short sequences of nearly equal weights: some results are small beside their terms."""
    b = 200
    lengths = [n] * b
    pool, g = pool_with(lengths, 1, 16, 48, cache_type, q_type, n)
    q = normal(g, b, 17, 48, dtype=q_type, scale=0.01)
    out, lse = KV.attend_token(q, pool.cache, pool.table, lens(lengths))
    check_token(pool, lengths, q, out, lse, None, 0)
