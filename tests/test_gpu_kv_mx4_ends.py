"""Attention over 4-bit values near the ends of f32: their sums stay finite while the maximum of the logits moves, and
small ones keep their bits."""
import numpy as np
import pytest
import torch

from gpu_helpers import require_gpu
from kv4_reference import Pool4
from shear_amd import kvcache as KV
from test_gpu_kvcache import BF16, check_prompt, check_token, lens, normal, prompt

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    return require_gpu()


@pytest.mark.parametrize("size", [2.5e38, 1e-22, 1e-36])
@pytest.mark.parametrize("how", ["level", "grow", "same"])
@pytest.mark.parametrize("page", [8, 16])
def test_values_near_the_ends(gpu, size, how, page):
    n, dim = 640, 64
    g = np.random.default_rng(7)
    q, k = normal(g, n, 2, dim), normal(g, n, 1, dim)
    if how == "grow":
        k = (k.float() * torch.linspace(0, 12, n, device="cuda")[:, None, None]).bfloat16()
    v = g.uniform(0.5, 1.0, (n, 1, dim)) * size
    if how != "same":
        v = v * g.choice([-1.0, 1.0], (n, 1, dim))
    pool = Pool4(1, -(-n // page), 1, page, dim, 3)
    pool.fill([n], k, torch.from_numpy(v).cuda())
    out, lse = prompt(pool, [n], [n], q)
    check_prompt(pool, [n], [n], q, out, lse, None, 0)
    for kw in ({}, {"weights": torch.zeros((1, 1, n), device="cuda")}):
        out, lse = KV.attend_token(q[-1:].contiguous(), pool.cache, pool.table, lens([n]), **kw)
        check_token(pool, [n], q[-1:], out, lse, None, 0)
