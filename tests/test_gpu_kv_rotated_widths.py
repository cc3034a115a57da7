"""The rotated append into codes where a row does not fill its lanes: the scale of a row is made of the row's dims alone,
whatever an earlier kernel left behind in the lanes' shared memory."""
import math

import numpy as np
import pytest
import torch

from gpu_helpers import require_gpu
from shear_amd import kvcache as KV
from test_gpu_kv_rotated import tokens_of
from test_gpu_kvcache import BF16, F16, SQ8, normal

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    return require_gpu()


def leave_behind(width, dtype, heads, kv):
    """Rows of ``width`` dims with weights of NaN, enough of them for every compute unit: all their factors are NaN."""
    n = 20000
    q, k = (torch.ones((n, h, width), dtype=dtype, device="cuda") for h in (heads, kv))
    w = torch.full((width,), math.nan, dtype=dtype, device="cuda")
    KV.append_rotated(KV.KvCache.allocate(1, kv, 1, width, dtype), q, k, k, torch.arange(n, dtype=torch.int32, device="cuda"),
                      torch.full((n,), -1, device="cuda"), KV.rotation_frequencies(width), w, w)


WIDTHS = [(16, 64, 2, 1), (32, 64, 4, 2), (48, 64, 1, 1), (80, 128, 8, 2), (96, 128, 5, 1), (112, 128, 16, 4), (144, 256, 2, 2),
          (160, 256, 4, 1), (192, 256, 8, 8)]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("kind,dim,width,heads,kv", [(SQ8, *w) for w in WIDTHS] + [(KV.MX4, *w) for w in WIDTHS if w[0] % 32 == 0])
@pytest.mark.parametrize("rotary,interleaved", [(16, False), ("all", False), ("all", True), (0, False)])
def test_lanes_past_the_row_add_nothing(gpu, dtype, kind, dim, width, heads, kv, rotary, interleaved):
    g = np.random.default_rng(dim)
    pages, page, n = 20, 16, 200
    q, k, v, positions, slots = tokens_of(g, n, heads, kv, dim, dtype, pages, page, 5000)
    rotary = dim if rotary == "all" else rotary
    f = KV.rotation_frequencies(rotary) if rotary else None
    w = normal(g, dim, dtype=dtype)
    plain, codes, again = (KV.KvCache.allocate(pages, kv, page, dim, t) for t in (dtype, kind, kind))
    for c in (codes, again):
        for t in c._tensors():
            t.view(torch.uint8).zero_()
    out = KV.append_rotated(plain, q, k, v, positions, slots, f, w, w, interleaved=interleaved)
    leave_behind(width, dtype, heads, kv)
    got = KV.append_rotated(codes, q, k, v, positions, slots, f, w, w, interleaved=interleaved)
    assert torch.equal(got, out) and out.isfinite().all()
    # the rounded rows, appended one by one where their slots say: the same codes and scales, to the bit
    rows = KV.read(plain, slots)
    KV.append(again, (slots // page).int()[:, None].contiguous(), (slots % page).int(), *rows)
    for x, y in zip(codes._tensors(), again._tensors()):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    assert KV.read(codes, slots)[0].isfinite().all()
