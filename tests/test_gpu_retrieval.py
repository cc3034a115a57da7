"""The cache, the graph search over its keys, the attention over what it finds and the
eviction, run together."""
import numpy as np
import pytest
import torch

from gpu_helpers import require_gpu
from shear_amd import kvcache as KV
from shear_amd import retrieval as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    return require_gpu()


def test_index_finds_the_largest_products(gpu):
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    keys = torch.randn((3000, 64), generator=g, device="cuda") * torch.rand((3000, 1), generator=g, device="cuda").add(0.5)
    q = torch.randn((50, 64), generator=g, device="cuda")
    got = R.KeyIndex(keys).search(q, 10, 100).cpu().numpy()
    want = (q @ keys.t()).topk(10, dim=1).indices.cpu().numpy()
    recall = np.mean([len(set(a) & set(b)) / 10 for a, b in zip(got.tolist(), want.tolist())])
    assert recall >= 0.9, recall


def test_distinct_rows(gpu):
    rows = torch.tensor([[5, -1, 5, 2], [7, 7, 7, 7]])
    assert R.distinct(rows).tolist() == [[-1, 2, 5, -1], [7, -1, -1, -1]]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.int8])
def test_context_end_to_end(gpu, dtype):
    got = R.run(rows=3000, tokens=4, keep=700, dtype=dtype)
    # fewer than a fifth of the rows are visible and carry most of the attention
    assert got["visible"] * 5 < 3004 and got["carried"] > 0.6
    assert got["kept"] == 700 and got["lengths"] == [704, 704] and got["finite"]


def test_token_sees_exactly_the_union(gpu):
    """The step's output is the attention over the first, the last and the found rows."""
    torch.manual_seed(1)
    c = R.LongContext(1, 2, 64, 1200, sinks=3, window=100, found=20, list_size=40)
    k, v = (torch.randn((1000, 2, 64), device="cuda").bfloat16() for _ in range(2))
    c.prompt(torch.randn((1000, 4, 64), device="cuda").bfloat16(), k, v, [1000])
    c.build()
    q = torch.randn((1, 4, 64), device="cuda").bfloat16()
    k1, v1 = (torch.randn((1, 2, 64), device="cuda").bfloat16() for _ in range(2))
    out = c.token(q, k1, v1)
    k, v = torch.cat([k, k1]).double(), torch.cat([v, v1]).double()
    for h in range(2):
        found = torch.cat([c.indexes[0][h].search(q[0, 2 * h: 2 * h + 2], 20, 40).flatten().long(),
                           torch.arange(3, device="cuda"), torch.arange(901, 1001, device="cuda")])
        rows = found[found >= 0].unique()
        p = torch.softmax(q[0, 2 * h: 2 * h + 2].double() @ k[rows, h].t() / 8, -1)
        want = p @ v[rows, h]
        # one rounding of the result and f32 arithmetic
        assert ((out[0, 2 * h: 2 * h + 2].double() - want).abs() <= 2**-8 * want.abs() + 1e-4).all()
        grown = c.weights[0, h].nonzero().squeeze(-1)
        assert torch.equal(grown, rows)
        assert torch.allclose(c.weights[0, h, rows].double(), p.sum(0), rtol=1e-5, atol=1e-9)
