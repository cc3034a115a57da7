"""4-bit caches on the GPU: rows stored and read to the bit, attention and eviction over them against 64-bit forms.
Unused slots of every cache are NaN."""
import math

import numpy as np
import pytest
import torch

from gpu_helpers import require_gpu
from kv4_reference import Pool4, mx4_rule, mx4_values
from kv_reference import attend, close
from shear_amd import kvcache as KV
from test_gpu_kvcache import BF16, F16, SQ8, check_prompt, check_token, kept_rows, lens, normal, pool_with, prompt

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    return require_gpu()


def pool4_with(lengths, heads, page, dim, q_type, seed, scale=1.0, **kw):
    g = np.random.default_rng(seed)
    pool = Pool4(len(lengths), max(1, -(-max(lengths) // page)), heads, page, dim, seed, **kw)
    total = int(sum(lengths))
    if total:
        pool.fill(lengths, *(normal(g, total, heads, dim, dtype=q_type, scale=scale) for _ in range(2)))
    return pool, g


def held(pool):
    """Values of the whole pool, keys and values."""
    kc, vc, ks, vs = (t.cpu().numpy() for t in pool.bytes())
    return [mx4_values(c, s) for c, s in ((kc, ks), (vc, vs))]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim,transposed,apart", [(32, False, 0), (64, False, 0), (96, True, 0), (128, False, 0),
                                                  (128, False, 3), (160, False, 0), (256, True, 0)])
def test_append(gpu, dtype, dim, transposed, apart):
    new, before, heads, page = [1, 0, 37, 64, 130], [5, 9, 0, 64, 3], 3, 16
    pool = Pool4(5, 9, heads, page, dim, dim, transposed=transposed, apart=apart)
    g = np.random.default_rng(dim)
    total = sum(new)
    # magnitudes from row to row, groups of zeros, a value that is alone in its group
    x = [g.standard_normal((total, heads, dim)) * 2.0 ** g.integers(-9, 9, (total, heads, 1)) for _ in range(2)]
    x[0][::5, :, :32] = 0.0
    x[1][::7, :, dim - 32:] *= np.arange(32) == 11
    k, v = (torch.from_numpy(y).to(dtype).cuda() for y in x)
    off = lens(np.concatenate([[0], np.cumsum(new)]).tolist())
    untouched = [t.clone() for t in pool.bytes()]
    KV.append(pool.cache, pool.table, lens(before), k, v, offsets=off, max_new=max(new))
    got = [t.cpu().numpy().copy() for t in pool.bytes()]
    at = 0
    for b, n in enumerate(new):
        rows = before[b] + np.arange(n)
        page_of, slot = pool.table_host[b][rows // page], rows % page
        for y, codes, scales in ((k, 0, 2), (v, 1, 3)):
            code, e = mx4_rule(y[at: at + n].double().cpu().numpy())
            assert np.array_equal(got[scales][page_of, :, slot], e), b
            there = got[codes][page_of, :, slot]
            have = np.stack([there & 15, there >> 4], -1).reshape(n, heads, dim)
            assert np.array_equal(have & 7, code & 7) and np.array_equal((have > 8) & (have != 8), (code > 8)), b
            # the rest of the pool is as it was
            got[codes][page_of, :, slot] = untouched[codes].cpu().numpy()[page_of, :, slot]
            got[scales][page_of, :, slot] = untouched[scales].cpu().numpy()[page_of, :, slot]
        at += n
    for a, b in zip(got, untouched):
        assert np.array_equal(a, b.cpu().numpy())


@pytest.mark.parametrize("dtype,mixed", [(BF16, False), (F16, False), (BF16, True), (F16, True)])
def test_append_values_of_every_size(gpu, dtype, mixed):
    """Every finite value of the type, the largest of its group or beside others; groups that are not finite."""
    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype).double().numpy()
    g = np.random.default_rng(5)
    if mixed:
        every = every[np.isfinite(every)]
        x = np.concatenate([g.permutation(every)[: len(every) // 64 * 64].reshape(-1, 64),
                            (np.sort(np.abs(every))[: len(every) // 64 * 64]).reshape(-1, 64)])
    else:
        x = every[:, None] * (g.random((65536, 64)) < 0.02)
        x[:, 5] = every
        x[:, 37] = every
        x = np.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0) + np.where(np.isfinite(every), 0, every)[:, None]
    n = len(x)
    pool = Pool4(1, -(-n // 256), 1, 256, 64, 3)
    k = torch.from_numpy(x).to(dtype).cuda().view(n, 1, 64)
    KV.append(pool.cache, pool.table, lens([0]), k, -k, offsets=lens([0, n]))
    code, e = mx4_rule(k.double().cpu().numpy())
    want = mx4_values(code[..., 0::2] | code[..., 1::2] << 4, e)
    keys, values, _ = pool.rows(0, n, 0)
    assert np.array_equal(keys, want[:, 0], equal_nan=True) and np.array_equal(values, -want[:, 0], equal_nan=True)


@pytest.mark.parametrize("dtype", [None, BF16, F16, torch.float32])
@pytest.mark.parametrize("dim,page,heads", [(32, 1, 1), (64, 16, 5), (96, 32, 2), (256, 64, 3), (128, 8, 8)])
def test_read(gpu, dtype, dim, page, heads):
    pool = Pool4(1, 9, heads, page, dim, 1, apart=dim % 3)
    pages = pool.cache.keys.shape[0]
    g = np.random.default_rng(2)
    kc, vc, ks, vs = pool.bytes()
    for t in (kc, vc):
        t.copy_(torch.from_numpy(g.integers(0, 256, t.shape, dtype=np.uint8)))
    for t in (ks, vs):  # every scale but those whose values pass f32's range
        t.copy_(torch.from_numpy(g.choice([*range(0, 253), 255], t.shape).astype(np.uint8)))
    keys, values = (torch.from_numpy(x) for x in held(pool))
    slots = g.integers(-3, pages * page + 3, 200)
    slots[:4] = [0, pages * page - 1, 2**40, -2**63]
    there = torch.from_numpy((slots >= 0) & (slots < pages * page))[:, None, None]
    at = np.where((slots >= 0) & (slots < pages * page), slots, 0)
    got = KV.read(pool.cache, torch.from_numpy(slots).cuda(), dtype)
    for x, pool_values in zip(got, (keys, values)):
        want = torch.where(there, pool_values[at // page, :, at % page], 0.0).to(dtype or BF16)
        assert x.dtype == (dtype or BF16) and x.shape == (200, heads, dim)
        assert torch.equal(x.cpu().nan_to_num(nan=3.0), want.nan_to_num(nan=3.0))
        assert torch.equal(x.isnan().cpu(), want.isnan())
    only, none = KV.read(pool.cache, torch.from_numpy(slots).cuda(), dtype, values=False)
    assert none is None and torch.equal(only.nan_to_num(nan=3.0), got[0].nan_to_num(nan=3.0))
    assert KV.read(pool.cache, torch.from_numpy(slots[:0]).cuda(), dtype)[0].shape == (0, heads, dim)


@pytest.mark.parametrize("cache_type", [BF16, F16, SQ8])
@pytest.mark.parametrize("dtype", [None, BF16, F16, torch.float32])
def test_read_of_the_other_types(gpu, cache_type, dtype):
    lengths = [70, 3]
    pool, _ = pool_with(lengths, 3, 16, 80, cache_type, F16 if cache_type == F16 else BF16, 4)
    own = torch.float32 if cache_type == SQ8 else cache_type
    for b, n in enumerate(lengths):
        rows = np.arange(n)
        slots = torch.from_numpy(pool.table_host[b][rows // 16].astype(np.int64) * 16 + rows % 16).cuda()
        k, v = KV.read(pool.cache, slots, dtype)
        for h in range(3):
            want_k, want_v, _ = pool.rows(b, n, h)
            for got, want in ((k, want_k), (v, want_v)):
                # (code * scale in f32, one rounding)
                assert torch.equal(got[:, h].cpu(), torch.from_numpy(want).float().to(dtype or own))


@pytest.mark.parametrize("q_type", [BF16, F16])
@pytest.mark.parametrize("dim,group,heads,page", [
    (64, 1, 3, 16), (128, 8, 2, 64), (96, 3, 2, 1), (32, 17, 1, 32), (256, 4, 1, 128), (160, 40, 1, 16), (224, 2, 2, 8)])
def test_token_all_rows(gpu, q_type, dim, group, heads, page):
    lengths = [0, 1, 2, 31, 32, 33, 127, 129, 700]
    pool, g = pool4_with(lengths, heads, page, dim, q_type, dim + group)
    q = normal(g, len(lengths), heads * group, dim, dtype=q_type, scale=2)
    out, lse = KV.attend_token(q, pool.cache, pool.table, lens(lengths))
    check_token(pool, lengths, q, out, lse, None, 0)


@pytest.mark.parametrize("q_type,dim", [(BF16, 64), (F16, 96), (BF16, 128), (F16, 256)])
@pytest.mark.parametrize("sinks,window", [(0, 1), (4, 100), (100, 0), (0, 0), (3, 5000), (64, 64)])
def test_token_window_list_and_weights(gpu, q_type, dim, sinks, window):
    lengths = [5, 0, 1000, 333, 64, 2500]
    pool, g = pool4_with(lengths, 2, 32, dim, q_type, 7 * sinks + window, apart=dim % 3)
    q = normal(g, len(lengths), 6, dim, dtype=q_type, scale=2)
    rows = np.full((len(lengths), 2, 77), -1, np.int32)
    for b, n in enumerate(lengths):
        for h in range(2):
            some = g.permutation(max(n, 1) + 9)[:60]  # distinct, some past the length
            rows[b, h, g.permutation(77)[: len(some)]] = some
    listed = torch.from_numpy(rows).cuda()
    weights = torch.zeros((len(lengths), 2, 2560), device="cuda")
    out, lse = KV.attend_token(q, pool.cache, pool.table, lens(lengths), sinks=sinks, window=window, listed=listed,
                               weights=weights)
    check_token(pool, lengths, q, out, lse, window, sinks, listed, weights)


@pytest.mark.parametrize("dim,group", [(128, 1), (128, 7), (64, 20), (256, 4)])
def test_token_weights_over_all_rows(gpu, dim, group):
    lengths = [9000, 3, 0, 300]
    pool, g = pool4_with(lengths, 2, 64, dim, BF16, group)
    q = normal(g, 4, 2 * group, dim, scale=2)
    weights = torch.zeros((4, 2, 9024), device="cuda")
    out, lse = KV.attend_token(q, pool.cache, pool.table, lens(lengths), weights=weights)
    check_token(pool, lengths, q, out, lse, None, 0, None, weights)


@pytest.mark.parametrize("q_type", [BF16, F16])
def test_token_pages_that_are_none_and_groups_that_are_nan(gpu, q_type):
    lengths = [300, 300, 300, 300]
    pool, g = pool4_with(lengths, 2, 16, 128, q_type, 3)
    pages = pool.cache.keys.shape[0]
    pool.table_host[0, 3:5] = -1
    pool.table_host[1, :] = pages  # past the last
    pool.table_host[2, 18] = 2**30
    pool.table = torch.from_numpy(pool.table_host).cuda()
    kc, vc, ks, vs = pool.bytes()
    vs[pool.table_host[3, 2], 1, 5, 2] = 255  # a value's dims 64..95
    ks[0], vs[0] = 255, 255  # what lies in row 0 of page 0 is read in the place of rows that are not there
    for b in range(4):
        pool.table_host[b][pool.table_host[b] == 0] = pages
    pool.table = torch.from_numpy(pool.table_host).cuda()
    q = normal(g, 4, 4, 128, dtype=q_type)
    out, lse = KV.attend_token(q, pool.cache, pool.table, lens(lengths))
    sub = [0, 1, 2]
    three = Pool4.__new__(Pool4)
    three.cache, three.table_host, three.page_rows = pool.cache, pool.table_host[:3], 16
    check_token(three, lengths[:3], q[sub], out[sub], lse[sub], None, 0)
    assert (out[1] == 0).all() and (lse[1] == -math.inf).all()
    nan = out[3].isnan().cpu()
    assert nan[2:, 64:96].all() and not nan[:2].any() and not nan[2:, :64].any() and not nan[2:, 96:].any()
    assert lse[3].isfinite().all()
    # a window without the row
    out, lse = KV.attend_token(q, pool.cache, pool.table, lens(lengths), sinks=30, window=200)
    assert out.isfinite().all()
    ks[pool.table_host[3, 18], 0, 11, 1] = 255  # a key of the last row: nothing is a number any more, of one head
    out, lse = KV.attend_token(q, pool.cache, pool.table, lens(lengths), sinks=30, window=200)
    assert out[3, :2].isnan().all() and lse[3, :2].isnan().all() and out[3, 2:].isfinite().all() and out[:3].isfinite().all()


@pytest.mark.parametrize("q_type", [BF16, F16])
def test_token_large_logits_and_scales_far_apart(gpu, q_type):
    """Rows whose scales lie 2^80 apart; fp16 queries meet scales that fp16 does not reach."""
    lengths, dim = [777, 40], 64
    pool, g = pool4_with(lengths, 2, 16, dim, BF16, 9)
    kc, vc, ks, vs = pool.bytes()
    shift = torch.from_numpy(g.integers(-40, 40, vs.shape)).cuda()
    vs.copy_((vs.long() + shift).clamp(2, 250).to(torch.uint8))
    ks.copy_((ks.long() + (shift > 37) * 3).clamp(2, 250).to(torch.uint8))
    q = normal(g, 2, 6, dim, dtype=q_type, scale=4)
    out, lse = KV.attend_token(q, pool.cache, pool.table, lens(lengths))
    qh, oh, lh = q.double().cpu().numpy(), out.double().cpu().numpy(), lse.double().cpu().numpy()
    for b, n in enumerate(lengths):
        for h in range(2):
            k, v, there = pool.rows(b, n, h)
            for i in range(3 * h, 3 * h + 3):
                want, z, _, spread, delta = attend(qh[b, i], k, v, there, 1 / math.sqrt(dim))
                fits = np.abs(want) < (6e4 if q_type == F16 else 3e38)
                assert close(oh[b, i], want, spread, delta, q_type, False)[fits].all()
                assert abs(lh[b, i] - z) <= delta + 2.0**-21 * (abs(z) + 1)


@pytest.mark.parametrize("q_type", [BF16, F16])
@pytest.mark.parametrize("group,dim", [(4, 64), (5, 128), (8, 256), (9, 64), (33, 32)])
def test_token_many_sequences(gpu, q_type, group, dim):
    """Lines of more sequences than a workgroup has threads, many of them short or empty, some pages missing."""
    g = np.random.default_rng(group)
    lengths = g.integers(0, 90, 300).tolist()
    lengths[5], lengths[100], lengths[299] = 2000, 0, 700
    pool, g = pool4_with(lengths, 1, 16, dim, q_type, 17)
    pool.table_host[5, 7] = pool.table_host[40] = -1
    pool.table_host[299, 40:42] = 10**9
    pool.table = torch.from_numpy(pool.table_host).cuda()
    q = normal(g, len(lengths), group, dim, dtype=q_type, scale=2)
    out, lse = KV.attend_token(q, pool.cache, pool.table, lens(lengths))
    check_token(pool, lengths, q, out, lse, None, 0)
    # lengths out of range: none, and clipped to max_length
    clipped = [-3 if n < 30 else 2**31 - 1 if n > 1000 else n for n in lengths]
    out, lse = KV.attend_token(q, pool.cache, pool.table, lens(clipped), max_length=1500)
    check_token(pool, [0 if n < 30 else min(n, 1500) for n in lengths], q, out, lse, None, 0)


@pytest.mark.parametrize("q_type", [BF16, F16])
def test_keys_and_values_of_different_layouts(gpu, q_type):
    lengths, heads, dim, page = [300, 77], 3, 96, 32
    pool, g = pool4_with(lengths, heads, page, dim, q_type, 19)
    c = pool.cache

    def other(t):  # rows first, room between them
        b = t.view(torch.uint8)
        wide = torch.full((b.shape[0], b.shape[2], b.shape[1], b.shape[3] + 16), 0xff, dtype=torch.uint8, device="cuda")
        y = wide[..., : b.shape[3]].transpose(1, 2)
        y.copy_(b)
        return y.view(t.dtype)

    mixed = KV.KvCache(c.keys, other(c.values), other(c.key_scales), c.value_scales)
    q, pq = normal(g, 2, 6, dim, dtype=q_type), normal(g, 150, 6, dim, dtype=q_type)
    w = [torch.zeros((2, heads, 320), device="cuda") for _ in range(2)]
    a = KV.attend_token(q, c, pool.table, lens(lengths), weights=w[0])
    b = KV.attend_token(q, mixed, pool.table, lens(lengths), weights=w[1])
    for x, y in zip((*a, w[0]), (*b, w[1])):
        assert torch.equal(x, y)
    for x, y in zip(KV.attend_prompt(pq, lens([0, 100, 150]), c, pool.table, lens(lengths)),
                    KV.attend_prompt(pq, lens([0, 100, 150]), mixed, pool.table, lens(lengths))):
        assert torch.equal(x, y)
    slots = torch.arange(c.keys.shape[0] * page, device="cuda")
    for x, y in zip(KV.read(c, slots), KV.read(mixed, slots)):
        assert torch.equal(x.nan_to_num(nan=9.0), y.nan_to_num(nan=9.0))
    k, v = normal(g, 2, heads, dim, dtype=q_type), normal(g, 2, heads, dim, dtype=q_type)
    for cache in (c, mixed):
        KV.append(cache, pool.table, lens([31, 5]), k, v)
    for x, y in zip(KV.read(c, slots), KV.read(mixed, slots)):
        assert torch.equal(x.nan_to_num(nan=9.0), y.nan_to_num(nan=9.0))
    kept = [KV.evict(cache, pool.table, lens(lengths), w[0], 50, sinks=2, recent=9) for cache in (c, mixed)]
    for x, y in zip(*kept):
        assert torch.equal(x, y)
    for x, y in zip(KV.read(c, slots), KV.read(mixed, slots)):
        assert torch.equal(x.nan_to_num(nan=9.0), y.nan_to_num(nan=9.0))


@pytest.mark.parametrize("q_type", [BF16, F16])
@pytest.mark.parametrize("group,page", [(3, 16), (3, 8), (8, 16), (20, 16)])
def test_queries_that_are_not_finite(gpu, q_type, group, page):
    """An infinite query times keys of one sign is an infinite logit of that sign: of minus infinity nothing is left."""
    lengths, dim = [200, 200, 200], 64
    pool, g = pool4_with(lengths, 1, page, dim, q_type, 13)
    kc, vc, ks, vs = pool.bytes()
    kc &= 0x77  # no key is negative
    kc |= 0x11  # or zero
    q = normal(g, 3, group, dim, dtype=q_type)
    q[0, 1, 5], q[1, 2, 7], q[2, 0, 40] = float("-inf"), float("inf"), float("nan")
    out, lse = KV.attend_token(q, pool.cache, pool.table, lens(lengths))
    assert (out[0, 1] == 0).all() and lse[0, 1] == -math.inf
    assert out[1, 2].isnan().all() and out[2, 0].isnan().all()
    rest = torch.ones((3, group), dtype=torch.bool, device="cuda")
    rest[0, 1] = rest[1, 2] = rest[2, 0] = False
    assert out[rest].isfinite().all() and lse[rest].isfinite().all()


def test_token_strides_and_transposed_pages(gpu):
    lengths = [100, 257]
    pool, g = pool4_with(lengths, 4, 32, 128, BF16, 11, transposed=True)
    wide = normal(g, 2, 16, 2, 128)
    q = wide[:, :, 1]
    out, lse = KV.attend_token(q, pool.cache, pool.table, lens(lengths), scale=1 / math.sqrt(128))
    check_token(pool, lengths, q, out, lse, None, 0)
    other = normal(g, 2, 8, 130)[:, :, 1:129]  # rows that are not 16-byte aligned
    out, lse = KV.attend_token(other, pool.cache, pool.table, lens(lengths))
    check_token(pool, lengths, other, out, lse, None, 0)


def test_past_32_bits(gpu):
    """A pool of 8 GiB of codes and one scale byte per 16 of them: rows and scales behind 4 GiB and 512 MiB."""
    pages, heads, page, dim = 2**17, 8, 128, 128
    c = KV.KvCache.allocate(pages, heads, page, dim, KV.MX4)
    last = [pages - 1, pages // 2 + 1, 3]
    table = torch.tensor([last], dtype=torch.int32, device="cuda")
    g = np.random.default_rng(3)
    n = 300
    k, v = normal(g, n, heads, dim), normal(g, n, heads, dim)
    KV.append(c, table, lens([0]), k, v, offsets=lens([0, n]))
    rows = np.arange(n)
    slots = torch.from_numpy(np.array(last, np.int64)[rows // page] * page + rows % page).cuda()
    for got, x in zip(KV.read(c, slots), (k, v)):
        code, e = mx4_rule(x.double().cpu().numpy())
        assert np.array_equal(got.double().cpu().numpy(), mx4_values(code[..., 0::2] | code[..., 1::2] << 4, e))
    small = KV.KvCache.allocate(3, heads, page, dim, KV.MX4)
    here = torch.arange(3, dtype=torch.int32, device="cuda")[None]
    KV.append(small, here, lens([0]), k, v, offsets=lens([0, n]))
    q = normal(g, 1, 16, dim)
    for a, b in zip(KV.attend_token(q, c, table, lens([n])), KV.attend_token(q, small, here, lens([n]))):
        assert torch.equal(a, b)
    q = normal(g, 70, 16, dim)
    for a, b in zip(KV.attend_prompt(q, lens([0, 70]), c, table, lens([n])),
                    KV.attend_prompt(q, lens([0, 70]), small, here, lens([n]))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("q_type", [BF16, F16])
@pytest.mark.parametrize("dim,group,heads,page", [
    (64, 1, 2, 16), (128, 4, 2, 64), (96, 3, 1, 8), (32, 7, 1, 32), (256, 2, 1, 128), (192, 1, 2, 1)])
def test_prompt_causal(gpu, q_type, dim, group, heads, page):
    new = [1, 0, 33, 200, 64, 5]
    lengths = [1, 40, 33, 263, 300, 700]
    pool, g = pool4_with(lengths, heads, page, dim, q_type, dim + group, apart=dim % 3)
    q = normal(g, sum(new), heads * group, dim, dtype=q_type, scale=2)
    out, lse = prompt(pool, lengths, new, q, max_new=200)
    check_prompt(pool, lengths, new, q, out, lse, None, 0)


@pytest.mark.parametrize("q_type,dim", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("sinks,window", [(0, 1), (4, 100), (70, 0), (0, 0), (0, 64), (200, 65), (5, 100000)])
def test_prompt_window_and_sinks(gpu, q_type, dim, sinks, window):
    new = [150, 1, 70]
    lengths = [600, 333, 70]
    pool, g = pool4_with(lengths, 2, 16, dim, q_type, window + sinks)
    q = normal(g, sum(new), 6, dim, dtype=q_type, scale=2)
    out, lse = prompt(pool, lengths, new, q, sinks=sinks, window=window)
    check_prompt(pool, lengths, new, q, out, lse, window, sinks)


@pytest.mark.parametrize("q_type,dim", [(BF16, 128), (F16, 128), (F16, 256)])
def test_prompt_few_tokens_over_a_long_cache(gpu, q_type, dim):
    lengths, new = [5000, 4100], [1, 3]  # split over the rows
    pool, g = pool4_with(lengths, 2, 64, dim, q_type, 8)
    q = normal(g, 4, 8, dim, dtype=q_type, scale=2)
    out, lse = prompt(pool, lengths, new, q)
    check_prompt(pool, lengths, new, q, out, lse, None, 0)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q_type", [BF16, F16])
def test_prompt_groups_that_are_nan_and_missing_pages(gpu, q_type, dim):
    """A value's group that only later queries see reaches those alone, in its dims; a key's likewise, in all."""
    n, page = 400, 16
    pool, g = pool4_with([n, n], 1, page, dim, q_type, 21)
    table = pool.table_host
    kc, vc, ks, vs = pool.bytes()
    vs[table[0, 350 // page], 0, 350 % page, 1] = 255
    ks[table[1, 360 // page], 0, 360 % page, 0] = 255
    pages = pool.cache.keys.shape[0]
    table[0, 2], table[1, 7] = -1, pages + 5
    pool.table = torch.from_numpy(table).cuda()
    q = normal(g, 2 * n, 3, dim, dtype=q_type, scale=2)
    out, lse = prompt(pool, [n, n], [n, n], q)
    first, second = out[:n].isnan(), out[n:].isnan()
    assert first[350:, :, 32:64].all() and not first[:350].any()
    assert not first[:, :, :32].any() and not first[:, :, 64:].any() and not lse[:n].isnan().any()
    assert second[360:].all() and not second[:360].any() and lse[n + 360:].isnan().all()
    # everything that is a number is the right one
    vs[table[0, 350 // page], 0, 350 % page, 1] = 120
    ks[table[1, 360 // page], 0, 360 % page, 0] = 120
    out, lse = prompt(pool, [n, n], [n, n], q)
    check_prompt(pool, [n, n], [n, n], q, out, lse, None, 0)


@pytest.mark.parametrize("q_type", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_scales_far_apart(gpu, q_type, dim):
    """Keys of small scales beside large ones, values 2^60 apart."""
    n = 200
    pool, g = pool4_with([n], 2, 16, dim, BF16, 31)
    kc, vc, ks, vs = pool.bytes()
    shift = torch.from_numpy(g.integers(-30, 30, vs.shape)).cuda()
    vs.copy_((vs.long() + shift).clamp(2, 250).to(torch.uint8))
    ks.copy_((ks.long() - shift.clamp(min=0)).clamp(2, 250).to(torch.uint8))
    q = normal(g, n, 4, dim, dtype=q_type, scale=2)
    out, lse = prompt(pool, [n], [n], q)
    qh, oh, lh = q.double().cpu().numpy(), out.double().cpu().numpy(), lse.double().cpu().numpy()
    for h in range(2):
        k, v, there = pool.rows(0, n, h)
        for i in range(0, n, 7):
            for a in range(2 * h, 2 * h + 2):
                want, z, _, spread, delta = attend(qh[i, a], k, v, np.arange(n) <= i, 1 / math.sqrt(dim))
                fits = np.abs(want) < (6e4 if q_type == F16 else 3e38)
                # fp16 queries: keys below 2^-24 of their row's largest scale are zeros
                delta += np.abs(qh[i, a]).sum() / math.sqrt(dim) * np.abs(k[: i + 1]).max() * 2.0**-24
                assert close(oh[i, a], want, spread, delta, q_type, True)[fits].all(), (i, a)
                assert abs(lh[i, a] - z) <= delta + 2.0**-21 * (abs(z) + 1)


def test_prompt_agrees_with_single_tokens(gpu):
    pool, g = pool4_with([500], 2, 32, 128, BF16, 51)
    q = normal(g, 500, 8, 128)
    out, lse = prompt(pool, [500], [500], q)
    for n in (1, 2, 64, 65, 300, 500):
        one, one_lse = KV.attend_token(q[n - 1: n], pool.cache, pool.table, lens([n]))
        assert torch.allclose(one.float(), out[n - 1: n].float(), atol=2e-2, rtol=2e-2)
        assert torch.allclose(one_lse, lse[n - 1: n], atol=1e-4, rtol=1e-5)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("dim,page,keep,sinks,recent,transposed,apart", [
    (64, 16, 100, 4, 20, False, 0), (128, 64, 700, 0, 0, True, 0), (256, 8, 33, 3, 30, False, 1),
    (96, 32, 1, 0, 1, False, 0), (32, 16, 257, 7, 50, False, 2)])
def test_evict(gpu, in_place, dim, page, keep, sinks, recent, transposed, apart):
    lengths, heads = [900, keep, 50, 0, 701], 2
    batch, columns = len(lengths), -(-900 // page)
    into_columns = -(-keep // page)
    pool, g = pool4_with(lengths, heads, page, dim, BF16, keep + dim, spare=batch * into_columns + 2,
                         transposed=transposed, apart=apart)
    pages = pool.cache.keys.shape[0]
    free = np.setdiff1d(np.arange(pages), pool.table_host.reshape(-1))
    into_host = g.permutation(free)[: batch * into_columns].reshape(batch, into_columns).astype(np.int32)
    into = None if in_place else torch.from_numpy(into_host).cuda()
    w = torch.from_numpy(np.exp(g.standard_normal((batch, heads, columns * page))).astype(np.float32)).cuda()
    was = [[pool.rows(b, n, h)[:2] for h in range(heads)] for b, n in enumerate(lengths)]
    kept, new_lengths, new_weights = KV.evict(pool.cache, pool.table, lens(lengths), w, keep, sinks=sinks, recent=recent,
                                              into=into)
    if not in_place:
        pool.table_host = into_host
    for b, n in enumerate(lengths):
        count = min(n, keep)
        assert int(new_lengths[b]) == count
        for h in range(heads):
            want = kept_rows(w[b, h].cpu().numpy(), n, keep, sinks, recent)
            assert np.array_equal(kept[b, h, :count].cpu().numpy(), want) and (kept[b, h, count:] == -1).all()
            k, v, _ = pool.rows(b, count, h)
            assert np.array_equal(k, was[b][h][0][want]) and np.array_equal(v, was[b][h][1][want])
            assert torch.equal(new_weights[b, h, :count].cpu(), w[b, h].cpu()[torch.from_numpy(np.asarray(want, np.int64))])


def test_stream_and_graph(gpu):
    lengths = [900, 100]
    pool, g = pool4_with(lengths, 2, 32, 128, BF16, 31)
    q = normal(g, 2, 8, 128)
    n = lens(lengths)
    want, want_lse = KV.attend_token(q, pool.cache, pool.table, n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got, lse = KV.attend_token(q, pool.cache, pool.table, n, stream=side)
    slots = torch.arange(64, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    rows = KV.read(pool.cache, slots, stream=side)[0]
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(lse, want_lse)
    assert torch.equal(rows.nan_to_num(nan=3.0), KV.read(pool.cache, slots)[0].nan_to_num(nan=3.0))
    weights = torch.zeros((2, 2, 928), device="cuda")
    k, v = normal(g, 2, 2, 128), normal(g, 2, 2, 128)
    off, pq = lens([0, 40, 50]), normal(g, 50, 8, 128)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        KV.append(pool.cache, pool.table, n - 1, k, v)
        out, lse = KV.attend_token(q, pool.cache, pool.table, n, weights=weights)
        asked, _ = KV.attend_prompt(pq, off, pool.cache, pool.table, n, max_new=40)
        kept, new, moved = KV.evict(pool.cache, pool.table, n, weights, 64, sinks=2, recent=8)
    for rep in range(3):
        weights.zero_()
        fill = [normal(np.random.default_rng(rep + i), 1000, 2, 128) for i in (0, 9)]
        pool.fill(lengths, *fill)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (out, lse, weights, asked, kept, new, moved)]
        pool.fill(lengths, *fill)
        KV.append(pool.cache, pool.table, n - 1, k, v)
        w = torch.zeros_like(weights)
        eager = [*KV.attend_token(q, pool.cache, pool.table, n, weights=w), w]
        eager.append(KV.attend_prompt(pq, off, pool.cache, pool.table, n, max_new=40)[0])
        eager += KV.evict(pool.cache, pool.table, n, w, 64, sinks=2, recent=8)
        torch.cuda.synchronize()
        for a, b in zip(got, eager):
            assert torch.equal(a, b), rep


def test_refusals(gpu):
    rows = torch.zeros((4, 2, 16, 32), dtype=torch.uint8, device="cuda").view(KV.MX4)
    scales = torch.zeros((4, 2, 16, 2), dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    for bad in (
            lambda: KV.KvCache(rows, rows),
            lambda: KV.KvCache(rows, rows, scales, scales[..., :1]),
            lambda: KV.KvCache(rows, rows, scales, scales.view(torch.uint8)),
            lambda: KV.KvCache(rows, rows, scales, scales.cpu()),
            lambda: KV.KvCache(rows, rows, torch.zeros((4, 2, 16), device="cuda"), torch.zeros((4, 2, 16), device="cuda")),
            lambda: KV.KvCache(rows, rows, scales, scales.view(torch.uint8).repeat(1, 1, 1, 2)[..., ::2].view(torch.float8_e8m0fnu)),
            lambda: KV.KvCache(rows.view(torch.uint8), rows.view(torch.uint8), scales, scales),
            lambda: KV.KvCache.allocate(4, 2, 16, 48, KV.MX4)):
        with pytest.raises(ValueError):
            bad()
    c = KV.KvCache(rows, rows.clone(), scales, scales.clone())
    assert c.head_dim == 64 and c.heads == 2 and c.page_rows == 16
    odd = torch.zeros((4, 2, 16, 24), dtype=torch.uint8, device="cuda").view(KV.MX4)  # 48 dims
    odd_scales = scales[..., :1]
    with pytest.raises(RuntimeError, match="multiple of 32"):
        KV.read(KV.KvCache(odd, odd, odd_scales, odd_scales), torch.zeros(1, dtype=torch.int64, device="cuda"))
    slots = torch.zeros(3, dtype=torch.int64, device="cuda")
    for bad in (lambda: KV.read(c, slots.int()), lambda: KV.read(c, slots[None]), lambda: KV.read(c, slots.cpu()),
                lambda: KV.read(c, slots, torch.float64), lambda: KV.read(c, slots, KV.MX4),
                lambda: KV.read(c, torch.zeros(6, dtype=torch.int64, device="cuda")[::2])):
        with pytest.raises(ValueError):
            bad()
    table, n = torch.zeros((1, 1), dtype=torch.int32, device="cuda"), lens([1])
    with pytest.raises(ValueError):
        KV.attend_token(torch.zeros((1, 2, 32), dtype=BF16, device="cuda"), c, table, n)  # the elements, not the dims
    with pytest.raises(ValueError):
        KV.append(c, table, n, torch.zeros((1, 2, 64), device="cuda"), torch.zeros((1, 2, 64), device="cuda"))
