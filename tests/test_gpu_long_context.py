"""A long context after its graphs were built, and at the end of its room."""
import pytest
import torch

from gpu_helpers import require_gpu
from shear_amd import retrieval as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    return require_gpu()


class Conversation:
    """A context of two heads of 64 dims and the rows that it should hold."""

    def __init__(self, seed, batch=1, **kw):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)
        self.c = R.LongContext(batch, 2, 64, **kw)
        self.batch = batch
        self.k = [torch.zeros((0, 2, 64), dtype=torch.float64, device="cuda") for _ in range(batch)]
        self.v = [torch.zeros((0, 2, 64), dtype=torch.float64, device="cuda") for _ in range(batch)]

    def normal(self, n, heads):
        return torch.randn((n, heads, 64), generator=self.g, device="cuda").bfloat16()

    def keep(self, k, v, new):
        for b, (x, y) in enumerate(zip(k.split(new), v.split(new))):
            self.k[b], self.v[b] = torch.cat([self.k[b], x.double()]), torch.cat([self.v[b], y.double()])

    def prompt(self, new):
        q, k, v = self.normal(sum(new), 4), self.normal(sum(new), 2), self.normal(sum(new), 2)
        self.c.prompt(q, k, v, new)
        self.keep(k, v, new)

    def token(self):
        """One step, checked against the attention over the first, the last, the found and the new rows."""
        c = self.c
        q, k, v = self.normal(self.batch, 4), self.normal(self.batch, 2), self.normal(self.batch, 2)
        before = c.weights.clone()
        out = c.token(q, k, v)
        self.keep(k, v, [1] * self.batch)
        for b in range(self.batch):
            n = self.k[b].shape[0]
            assert int(c.lengths[b]) == n
            for h in range(2):
                rows = torch.arange(n, device="cuda")
                if c.indexes:
                    found = c.indexes[b][h].search(q[b, 2 * h: 2 * h + 2], c.found, c.list_size).flatten().long()
                    since = n - c.shown()
                    assert since <= self.built[b]
                    rows = torch.cat([found[found >= 0], rows[: c.sinks], rows[since:]]).unique()
                p = torch.softmax(q[b, 2 * h: 2 * h + 2].double() @ self.k[b][rows, h].t() / 8, -1)
                want = p @ self.v[b][rows, h]
                # one rounding of the result and f32 arithmetic
                assert ((out[b, 2 * h: 2 * h + 2].double() - want).abs() <= 2**-8 * want.abs() + 1e-4).all(), (b, h)
                grown = (c.weights[b, h] != before[b, h]).nonzero().squeeze(-1)
                assert set(grown.tolist()) <= set(rows.tolist()) and n - 1 in grown
        return out

    def build(self):
        self.c.build()
        self.built = [x.shape[0] for x in self.k]


def test_a_second_prompt_is_seen(gpu):
    t = Conversation(1, batch=2, max_rows=1500, sinks=3, window=50, found=20, list_size=40)
    t.prompt([700, 640])
    t.build()
    t.token()
    t.prompt([300, 10])  # far more than the window
    weights = t.c.weights.clone()
    t.token()
    gained = t.c.weights - weights
    assert (gained[0, :, 700:1002] > 0).all()  # every row that is in no graph
    t.build()
    t.token()


def test_more_tokens_than_the_window(gpu):
    t = Conversation(2, max_rows=800, sinks=2, window=8, found=10, list_size=20)
    t.prompt([600])
    t.build()
    for _ in range(20):
        t.token()
    t.build()
    t.token()


@pytest.mark.parametrize("page_rows", [64, 16])
def test_no_room_is_refused(gpu, page_rows):
    t = Conversation(3, batch=2, max_rows=200, page_rows=page_rows, sinks=2, window=20)
    t.prompt([198, 150])
    for new, tokens in (([3, 0], 3), ([0, 51], 51), ([1], 1), ([1, -1], 0), ([1, 1], 3)):
        q, k, v = t.normal(tokens, 4), t.normal(tokens, 2), t.normal(tokens, 2)
        with pytest.raises(ValueError):
            t.c.prompt(q, k, v, new)
            pytest.fail(f"{new} was not refused")
    t.prompt([1, 1])
    t.token()  # the last row of the first
    lengths, keys = t.c.lengths.clone(), t.c.cache.keys.clone()
    with pytest.raises(ValueError, match="room"):
        t.c.token(t.normal(2, 4), t.normal(2, 2), t.normal(2, 2))
    assert torch.equal(t.c.lengths, lengths) and torch.equal(t.c.cache.keys.view(torch.int16), keys.view(torch.int16))
    kept = t.c.evict(100)
    assert t.c.lengths.tolist() == [100, 100]
    for b in range(2):  # (both heads' own rows)
        at = kept[b].long().t().unsqueeze(-1).expand(-1, -1, 64)
        t.k[b], t.v[b] = t.k[b].gather(0, at), t.v[b].gather(0, at)
    t.token()
    t.prompt([99, 1])
