"""The key-value cache's Python calls: what they refuse."""
import pytest
import torch

from gpu_helpers import require_gpu
from shear_amd import kvcache as KV
from test_gpu_kvcache import BF16, lens, normal, pool_with

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    return require_gpu()


def test_tensors_that_require_a_gradient_are_refused(gpu):
    pool, g = pool_with([40, 20], 2, 16, 64, BF16, BF16, 1)
    c, t, n = pool.cache, pool.table, lens([40, 20])
    q, k, v = normal(g, 2, 4, 64), normal(g, 2, 2, 64), normal(g, 2, 2, 64)
    w = torch.ones((2, 2, 48), device="cuda")

    def needs(x):
        return x.detach().clone().requires_grad_()

    grown = KV.KvCache(needs(c.keys), c.values)
    calls = [
        lambda: KV.attend_token(needs(q), c, t, n),
        lambda: KV.attend_token(q, c, t, n, weights=needs(w)),
        lambda: KV.attend_token(q, grown, t, n),
        lambda: KV.attend_prompt(needs(q), lens([0, 1, 2]), c, t, n),
        lambda: KV.append(c, t, n - 1, needs(k), v),
        lambda: KV.append(c, t, n - 1, k, needs(v)),
        lambda: KV.append(grown, t, n - 1, k, v),
        lambda: KV.evict(c, t, n, needs(w), 8),
        lambda: KV.evict(grown, t, n, w, 8),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError, match="gradient"):
            call()
            pytest.fail(f"call {i} was not refused")
    want = KV.attend_token(q, c, t, n)
    with torch.no_grad():
        got = KV.attend_token(needs(q), c, t, n)
        calls[-1]()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and not got[0].requires_grad


def test_tensors_without_dimensions_are_refused(gpu):
    pool, g = pool_with([40, 20], 2, 16, 64, BF16, BF16, 1)
    c, t, n = pool.cache, pool.table, lens([40, 20])
    q, k = normal(g, 2, 4, 64), normal(g, 2, 2, 64)
    w = torch.ones((2, 2, 48), device="cuda")
    calls = [
        lambda: KV.attend_prompt(q[0, 0, 0], lens([0, 1, 2]), c, t, n),
        lambda: KV.attend_prompt(q, lens([0, 1, 2]), c, t[0, 0], n),
        lambda: KV.attend_prompt(q, lens([0, 1, 2])[0], c, t, n),
        lambda: KV.attend_token(q[0, 0, 0], c, t, n),
        lambda: KV.attend_token(q, c, t[0, 0], n),
        lambda: KV.attend_token(q, c, t, n[0]),
        lambda: KV.attend_token(q, c, t, n, weights=w[0, 0, 0]),
        lambda: KV.append(c, t, n, k[0, 0, 0], k[0, 0, 0]),
        lambda: KV.append(c, t[0, 0], n, k, k),
        lambda: KV.evict(c, t, n, w[0, 0, 0], 8),
        lambda: KV.evict(c, t, n, w, 8, into=t[0, 0]),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
