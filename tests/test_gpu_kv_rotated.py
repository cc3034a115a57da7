"""The rotated append (kvcache.append_rotated) against 64-bit forms, and against append where rows are codes."""
import numpy as np
import pytest
import torch

from gpu_helpers import require_gpu
from kv4_reference import rotated
from kv_reference import ROUND
from shear_amd import kvcache as KV
from test_gpu_kvcache import BF16, F16, SQ8, normal

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    return require_gpu()


def near(got, want, size, dtype):
    """One rounding, and in f32: the sum of squares and its root (7 + 4 units in the last place), two products, the sine's
    2^-22.5 and three operations of the rotation, together less than 2^-19 of the pair's values."""
    u = ROUND[dtype]
    tol = 2.0**-126 + u * np.abs(want) + (1 + u) * 2.0**-19 * size + (2.0**-25 if dtype == F16 else 0.0)
    return np.abs(got - want) <= tol * 1.01


def tokens_of(g, n, heads, kv, dim, dtype, pages, page, far):
    q, k, v = (normal(g, n, h, dim, dtype=dtype, scale=3) for h in (heads, kv, kv))
    positions = torch.from_numpy(g.integers(0, far, n).astype(np.int32)).cuda()
    slots = torch.from_numpy(g.permutation(pages * page)[:n].astype(np.int64)).cuda()
    return q, k, v, positions, slots


def check(cache, q, k, v, positions, slots, frequencies, wq, wk, eps, interleaved, out, keys_before, values_before):
    page, pages = cache.page_rows, cache.keys.shape[0]
    p, s = positions.cpu().numpy(), slots.cpu().numpy()
    f = None if frequencies is None else frequencies.cpu().numpy()
    weights = [None if w is None else w.double().cpu().numpy() for w in (wq, wk)]
    real = p >= 0
    want, size = rotated(q.double().cpu().numpy(), p, f, weights[0], eps, interleaved)
    got = out.double().cpu().numpy()
    assert near(got[real], want[real], size[real], q.dtype).all()
    assert (got[~real] == 0).all()
    want, size = rotated(k.double().cpu().numpy(), p, f, weights[1], eps, interleaved)
    written = real & (s >= 0) & (s < pages * page)
    at = s[written]
    got = cache.keys.double().cpu().numpy()[at // page, :, at % page]
    assert near(got, want[written], size[written], q.dtype).all()
    at = torch.from_numpy(at).cuda()
    keys, values = keys_before.clone(), values_before.clone()
    keys[at // page, :, at % page] = cache.keys[at // page, :, at % page]
    values[at // page, :, at % page] = v[torch.from_numpy(written).cuda()]
    assert torch.equal(cache.keys, keys) and torch.equal(cache.values, values)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim,heads,kv,rotary,interleaved,norm", [
    (128, 8, 2, 128, False, "both"), (64, 3, 3, 64, True, "both"), (80, 5, 1, 80, False, "q"), (96, 4, 2, 32, False, "k"),
    (256, 2, 1, 256, False, "f32"), (16, 1, 1, 16, False, "both"), (128, 40, 8, 64, True, "none"), (192, 2, 2, 0, False, "both"),
    (32, 1, 1, 16, True, "f32"), (128, 1, 64, 128, False, "none"), (64, 7, 2, 0, False, "none"), (256, 33, 1, 208, True, "both")])
@pytest.mark.parametrize("n", [1, 7, 150])
def test_rows(gpu, dtype, dim, heads, kv, rotary, interleaved, norm, n):
    g = np.random.default_rng(dim + heads + n)
    pages, page = 30, 16
    cache = KV.KvCache(*(normal(g, pages, kv, page, dim, dtype=dtype) for _ in range(2)))
    before = cache.keys.clone(), cache.values.clone()
    q, k, v, positions, slots = tokens_of(g, n, heads, kv, dim, dtype, pages, page, 100000)
    f = KV.rotation_frequencies(rotary) if rotary else None
    w = [(1 + normal(g, dim, dtype=torch.float32, scale=0.3)).to(torch.float32 if norm == "f32" else dtype) for _ in range(2)]
    wq = w[0] if norm in ("both", "q", "f32") else None
    wk = w[1] if norm in ("both", "k", "f32") else None
    out = KV.append_rotated(cache, q, k, v, positions, slots, f, wq, wk, eps=1e-5, interleaved=interleaved)
    check(cache, q, k, v, positions, slots, f, wq, wk, 1e-5, interleaved, out, *before)


@pytest.mark.parametrize("interleaved", [False, True])
def test_positions_padding_and_slots_that_are_none(gpu, interleaved):
    g = np.random.default_rng(1)
    pages, page, dim = 5, 32, 128
    cache = KV.KvCache(*(normal(g, pages, 2, page, dim) for _ in range(2)))
    before = cache.keys.clone(), cache.values.clone()
    q, k, v, positions, slots = tokens_of(g, 60, 6, 2, dim, BF16, pages, page, 2**30)
    positions[:8] = torch.tensor([0, 1, -1, -2**31, 2**30 - 1, 2**31 - 1, 10**6, 131071], dtype=torch.int32)
    slots[8:13] = torch.tensor([-1, -2**63, pages * page, 2**32, 2**62], dtype=torch.int64)
    f = KV.rotation_frequencies(dim, base=500000.0)
    w = normal(g, dim)
    out = KV.append_rotated(cache, q, k, v, positions, slots, f, w, w, interleaved=interleaved)
    check(cache, q, k, v, positions, slots, f, w, w, 1e-6, interleaved, out, *before)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("kind", [SQ8, KV.MX4])
@pytest.mark.parametrize("dim,heads,kv", [(128, 8, 2), (64, 4, 4), (96, 5, 1), (256, 2, 2), (32, 1, 3)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_codes_are_those_of_the_rounded_rows(gpu, dtype, kind, dim, heads, kv, interleaved):
    g = np.random.default_rng(dim)
    pages, page, n = 20, 16, 200
    q, k, v, positions, slots = tokens_of(g, n, heads, kv, dim, dtype, pages, page, 5000)
    k[3, 0, 5], v[9, kv - 1, 7] = float("nan"), float("inf")
    positions[20:25] = -1
    f, w = KV.rotation_frequencies(dim // 32 * 32), normal(g, dim, dtype=dtype)
    plain, codes, again = (KV.KvCache.allocate(pages, kv, page, dim, t) for t in (dtype, kind, kind))
    for c in (codes, again):
        for t in c._tensors():
            t.view(torch.uint8).zero_()
    a, b = (KV.append_rotated(c, q, k, v, positions, slots, f, w, w, interleaved=interleaved) for c in (plain, codes))
    assert torch.equal(a, b)
    # the rounded rows, appended one by one where their slots say
    real = (positions >= 0).nonzero().squeeze(-1)
    at = slots[real]
    rows = KV.read(plain, at)
    KV.append(again, (at // page).int()[:, None].contiguous().repeat(1, 1), (at % page).int(), *rows)
    for x, y in zip(codes._tensors(), again._tensors()):
        x, y = x.view(torch.uint8), y.view(torch.uint8)
        assert torch.equal(x, y)


def test_values_that_are_not_finite_and_rows_of_zeros(gpu):
    g = np.random.default_rng(4)
    cache = KV.KvCache.allocate(2, 1, 16, 64)
    q, k, v, positions, slots = tokens_of(g, 8, 2, 1, 64, BF16, 2, 16, 100)
    q[1] = 0
    q[2, 0, 5], q[3, 1, 7], v[4, 0, 3] = float("nan"), float("inf"), float("-inf")
    w = torch.ones(64, dtype=BF16, device="cuda")
    out = KV.append_rotated(cache, q, k, v, positions, slots, KV.rotation_frequencies(64), w, w)
    assert (out[1] == 0).all() and out[2, 0].isnan().all() and out[3, 1, [7, 39]].isnan().all()
    rest = out.clone()
    rest[2, 0] = rest[3, 1] = 0
    assert rest.isfinite().all()  # no other row
    got = KV.read(cache, slots)[1]
    assert torch.equal(got, v)


def test_strides_streams_and_graph(gpu):
    g = np.random.default_rng(2)
    pages, page, dim, n = 40, 16, 128, 90
    qkv = normal(g, n, 12, dim)  # one product's rows, as a layer gives them
    q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
    positions = torch.arange(n, dtype=torch.int32, device="cuda")
    slots = torch.from_numpy(g.permutation(pages * page)[:n].astype(np.int64)).cuda()
    f, w = KV.rotation_frequencies(dim), normal(g, dim)
    caches = [KV.KvCache(torch.zeros((pages, page, 2, dim), dtype=BF16, device="cuda").transpose(1, 2),
                         torch.zeros((pages, 2, page, dim), dtype=BF16, device="cuda")) for _ in range(3)]
    before = caches[0].keys.clone(), caches[0].values.clone()
    out = KV.append_rotated(caches[0], q, k, v, positions, slots, f, w, None)
    check(caches[0], q, k, v, positions, slots, f, w, None, 1e-6, False, out, *before)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    # rows that are not 16-byte aligned are copied, on the stream
    odd = normal(g, n, 8, dim + 1)[..., 1:]
    odd.copy_(q)
    side.wait_stream(torch.cuda.current_stream())
    got = KV.append_rotated(caches[1], odd, k.contiguous(), v, positions, slots, f, w, None, stream=side)
    side.synchronize()
    assert torch.equal(got, out) and torch.equal(caches[1].keys, caches[0].keys)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        replayed = KV.append_rotated(caches[2], q, k, v, positions, slots, f, w, w)
    for seed in range(3):
        qkv.copy_(normal(np.random.default_rng(seed), n, 12, dim))
        positions.add_(1000)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        a = replayed.clone(), caches[2].keys.clone()
        want = KV.append_rotated(caches[1], q, k, v, positions, slots, f, w, w)
        assert torch.equal(a[0], want) and torch.equal(a[1], caches[1].keys)


def test_more_rows_than_a_workgroup_and_many_tokens(gpu):
    g = np.random.default_rng(6)
    n, pages, page = 3001, 200, 16
    cache = KV.KvCache(*(normal(g, pages, 4, page, 64) for _ in range(2)))
    before = cache.keys.clone(), cache.values.clone()
    q, k, v, positions, slots = tokens_of(g, n, 5, 4, 64, BF16, pages, page, 3000000)
    f = KV.rotation_frequencies(64)
    out = KV.append_rotated(cache, q, k, v, positions, slots, f)
    check(cache, q, k, v, positions, slots, f, None, None, 1e-6, False, out, *before)


def test_refusals(gpu):
    g = np.random.default_rng(1)
    cache = KV.KvCache.allocate(2, 2, 16, 64)
    q, k, v, positions, slots = tokens_of(g, 3, 4, 2, 64, BF16, 2, 16, 9)
    f, w = KV.rotation_frequencies(64), normal(g, 64)
    good = dict(cache=cache, q=q, k=k, v=v, positions=positions, slots=slots, frequencies=f, q_weight=w, k_weight=w)
    KV.append_rotated(**good)
    assert KV.append_rotated(**{**good, "q": q[:0], "k": k[:0], "v": v[:0], "positions": positions[:0], "slots": slots[:0]}).shape == (0, 4, 64)
    for change in (dict(q=q.float()), dict(q=q.half()), dict(q=q[0]), dict(q=q[..., :48]), dict(q=q[:, :0]), dict(q=q.cpu()),
                   dict(k=k[:2]), dict(k=k.half()), dict(v=v[:, :1]), dict(positions=positions.long()),
                   dict(positions=positions[:2]), dict(slots=slots.int()), dict(slots=slots[:2]), dict(slots=slots[0]),
                   dict(frequencies=f.float()), dict(frequencies=f[:4]), dict(frequencies=KV.rotation_frequencies(80)),
                   dict(q_weight=w.half()), dict(q_weight=w[:32]), dict(k_weight=w.float()), dict(eps=-1.0),
                   dict(eps=float("nan")), dict(q=q.detach().requires_grad_()), dict(k=k.detach().requires_grad_()),
                   dict(q_weight=w.detach().requires_grad_()),
                   dict(frequencies=f.clone().requires_grad_())):
        with pytest.raises(ValueError):
            KV.append_rotated(**{**good, **change})
            pytest.fail(f"{change} was not refused")
