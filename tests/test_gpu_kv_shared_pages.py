"""Sequences whose tables name the same pages (a prompt in common): every operator that reads gives what it gives over pages of
their own, to the bit."""
import numpy as np
import pytest
import torch

from gpu_helpers import require_gpu
from shear_amd import kvcache as KV
from test_gpu_kvcache import BF16, F16, SQ8, lens, normal

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    return require_gpu()


@pytest.mark.parametrize("kind,q_type", [(KV.MX4, BF16), (KV.MX4, F16), (SQ8, BF16), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("group,dim", [(2, 64), (8, 128), (20, 64), (4, 256)])
def test_a_prompt_in_common(gpu, kind, q_type, group, dim):
    batch, page, common, heads = 9, 16, 20, 2
    g = np.random.default_rng(group)
    lengths = [common * page + n for n in (1, 0, 15, 16, 17, 100, 33, 64, 5)]
    columns = common + 7
    own = KV.KvCache.allocate(batch * columns, heads, page, dim, kind)
    table = torch.from_numpy(g.permutation(batch * columns).reshape(batch, columns).astype(np.int32)).cuda()
    shared = table.clone()
    shared[:, :common] = table[4, :common]
    k, v = (normal(g, common * page, heads, dim, dtype=q_type) for _ in range(2))
    for b in range(batch):  # the same rows in everyone's own pages
        KV.append(own, table[b: b + 1], lens([0]), k, v, offsets=lens([0, common * page]))
        rest = lengths[b] - common * page
        if rest:
            KV.append(own, table[b: b + 1], lens([common * page]), *(normal(g, rest, heads, dim, dtype=q_type) for _ in range(2)),
                      offsets=lens([0, rest]))
    n, rows = lens(lengths), columns * page
    q, pq = normal(g, batch, heads * group, dim, dtype=q_type), normal(g, 3 * batch, heads * group, dim, dtype=q_type)
    off = lens(range(0, 3 * batch + 1, 3))
    listed = torch.arange(200, 240, dtype=torch.int32, device="cuda").expand(batch, heads, 40).contiguous()
    got = []
    for t in (table, shared):
        weights = [torch.zeros((batch, heads, rows), device="cuda") for _ in range(2)]
        got.append([*KV.attend_token(q, own, t, n), *KV.attend_token(q, own, t, n, weights=weights[0]),
                    *KV.attend_token(q, own, t, n, sinks=4, window=50, listed=listed, weights=weights[1]), *weights,
                    *KV.attend_prompt(pq, off, own, t, n), *KV.attend_prompt(pq, off, own, t, n, sinks=4, window=100)])
    for x, y in zip(*got):
        assert torch.equal(x, y)
