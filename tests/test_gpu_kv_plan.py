"""The plan of a step (kvcache.plan) against the rule written out on the host."""
import numpy as np
import pytest
import torch

import kv4_reference as R
from gpu_helpers import require_gpu
from shear_amd import kvcache as KV

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    return require_gpu()


def dev(x, dtype=torch.int32):
    return torch.as_tensor(np.asarray(x), dtype=dtype, device="cuda")


def check(page, table, lengths, held, new, free, count, tokens, stream=None, wide=0):
    t, f = dev(np.pad(table, ((0, 0), (0, wide)), constant_values=-7)), dev(free)
    view = t[:, : table.shape[1]] if wide else t
    got = KV.plan(page, view, dev(lengths), dev(held), dev(new), f, dev([count]), tokens, stream=stream)
    want = R.plan(page, table, lengths, held, new, free, count, tokens)
    torch.cuda.synchronize()
    names = ("lengths", "held", "count", "granted", "offsets", "positions", "sequences", "slots")
    for name, x in zip(names, want):
        y = getattr(got, name)
        assert y.dtype == (torch.int64 if name == "slots" else torch.int32)
        assert np.array_equal(y.cpu().numpy(), np.minimum(x, 2**31 - 1) if name == "offsets" else x), name
    assert np.array_equal(view.cpu().numpy(), want[8]) and np.array_equal(f.cpu().numpy(), want[9])
    if wide:
        assert (t[:, table.shape[1]:] == -7).all()
    return got, want


def drawn(g, batch, columns, page, spare, new_most, ends=0.1):
    """A consistent state: pages held by nobody twice, some sequences with more than they need."""
    held = g.integers(0, columns + 1, batch)
    lengths = np.array([g.integers(max(0, (h - 2) * page), h * page + 1) for h in held])
    new = np.where(g.random(batch) < ends, -1, g.integers(0, new_most + 1, batch))
    used = int(held.sum())
    ids = g.permutation(used + spare).astype(np.int32)
    table, at = np.full((batch, columns), -1, np.int32), 0
    for b in range(batch):
        table[b, : held[b]] = ids[at: at + held[b]]
        at += held[b]
    free = np.full(used + spare, -9, np.int32)
    free[:spare] = ids[used:]
    return table, lengths.astype(np.int32), held.astype(np.int32), new.astype(np.int32), free


@pytest.mark.parametrize("batch,columns,page,spare,new_most", [
    (1, 1, 1, 0, 1), (1, 40, 16, 60, 500), (5, 3, 65536, 4, 100000), (64, 20, 16, 1000, 1), (200, 64, 16, 300, 90),
    (1023, 5, 8, 900, 20), (1024, 5, 8, 5000, 20), (1025, 5, 8, 0, 20), (5000, 3, 4, 3000, 5), (3, 700, 1, 900, 600),
    (0, 4, 16, 8, 1), (7, 0, 16, 3, 2)])
def test_drawn_steps(gpu, batch, columns, page, spare, new_most):
    for seed in range(3):
        g = np.random.default_rng(seed)
        table, lengths, held, new, free = drawn(g, batch, columns, page, spare, new_most)
        total = int(np.maximum(new, 0).sum())
        for tokens in {total, total + 37, total // 2, 0}:
            check(page, table, lengths, held, new, free, spare, tokens, wide=seed)


def test_padding_and_steps_that_follow_each_other(gpu):
    """What one step gives is what the next takes; no page is ever in two places."""
    g = np.random.default_rng(7)
    batch, columns, page, pages = 37, 12, 16, 300
    table, free = np.full((batch, columns), -1, np.int32), np.arange(pages, dtype=np.int32)[::-1].copy()
    lengths, held, count = np.zeros(batch, np.int32), np.zeros(batch, np.int32), pages
    for step in range(30):
        new = np.where(g.random(batch) < 0.07, -1, np.where(g.random(batch) < 0.2, g.integers(0, 120, batch), 1)).astype(np.int32)
        got, want = check(page, table, lengths, held, new, free, count, int(np.maximum(new, 0).sum()) + 5)
        lengths, held, count = np.array(want[0], np.int32), np.array(want[1], np.int32), want[2][0]
        table, free = want[8], want[9]
        own = np.concatenate([table[b, : held[b]] for b in range(batch)] + [free[:count]])
        assert np.array_equal(np.sort(own), np.arange(pages))
        real = want[7][want[7] >= 0]
        assert len(np.unique(real)) == len(real)


def test_too_few_pages_and_who_is_served(gpu):
    """One that needs none is served behind one that is not; one that needs pages behind it is not."""
    table = np.arange(12, dtype=np.int32).reshape(4, 3)
    free = np.array([12, 13, 0, 0], np.int32)
    got, _ = check(4, table, np.array([4, 3, 4, 8]), np.array([1, 1, 1, 2]), np.array([9, 1, 1, 0]), free, 2, 11)
    # 13 rows would pass the table of the first: what it would need does not count
    assert got.granted.tolist() == [0, 1, 1, 0] and got.lengths.tolist() == [4, 4, 5, 8]
    got, _ = check(4, table, np.array([4, 3, 4, 8]), np.array([1, 1, 1, 2]), np.array([8, 1, 1, 0]), free, 1, 10)
    assert got.granted.tolist() == [0, 1, 0, 0] and got.lengths.tolist() == [4, 4, 4, 8] and got.count.tolist() == [1]
    got, _ = check(4, table, np.array([4, 3, 4, 8]), np.array([1, 1, 1, 2]), np.array([8, 1, 1, -3]), free, 2, 10)
    assert got.granted.tolist() == [8, 1, 1, 0] and got.count.tolist() == [1] and got.held.tolist() == [3, 1, 2, 0]


def test_numbers_that_make_no_sense(gpu):
    """Lengths, held pages and counts out of range are clipped, ids that name no page give no place."""
    g = np.random.default_rng(3)
    table = g.integers(-2**31, 2**31 - 1, (6, 4), dtype=np.int64).astype(np.int32)
    free = np.array([5, -1, 7, 2**31 - 1, -2**31, 1], np.int32)
    big = 2**31 - 1
    for count in (-5, 0, 3, 6, big):
        check(16, table, np.array([-1, big, 64, 3, -big, 10]), np.array([big, -4, 2, 0, 4, 4]),
              np.array([5, 1, 0, big, 2, -big]), free, count, 40)
    # sums past 32 bits: nothing past the tokens is granted
    check(16, table, np.zeros(6, np.int32), np.full(6, 4), np.full(6, big), free, 2, 100)


def test_tables_past_32_bits_and_places_past_32_bits(gpu):
    columns, page = 40000, 65536  # 2.6e9 rows: sequences end at 2^30 - 1
    table = np.full((2, columns), 3, np.int32)
    table[1, 16383] = 2**20
    lengths = np.array([2**30 - 3, 2**30 - 20], np.int32)
    held = np.array([16384, 16384], np.int32)
    got, _ = check(page, table, lengths, held, np.array([3, 19]), np.zeros(1, np.int32), 0, 22)
    assert got.granted.tolist() == [0, 19] and int(got.slots.max()) == 2**20 * 65536 + 65534


def test_many_tokens(gpu):
    g = np.random.default_rng(5)
    for batch in (3, 6000):
        table, lengths, held, new, free = drawn(g, batch, 400 if batch == 3 else 4, 16, 3000, 5000 if batch == 3 else 7)
        check(16, table, lengths, held, new, free, 3000, int(np.maximum(new, 0).sum()) + 1)


def test_stream_and_graph(gpu):
    g = np.random.default_rng(9)
    table, lengths, held, new, free = drawn(g, 100, 10, 16, 200, 70)
    total = int(np.maximum(new, 0).sum())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    check(16, table, lengths, held, new, free, 200, total, stream=side)
    for tokens in (total, 6000):
        args = [dev(x) for x in (table, lengths, held, new, free, [200])]
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            got = KV.plan(16, *args, tokens)
        for seed in range(3):
            state = drawn(np.random.default_rng(seed), 100, 10, 16, 200, 50)
            for a, x in zip(args, (*state[:4], np.resize(state[4], len(free)), [150])):
                a.copy_(dev(x))
            want = R.plan(16, *state[:4], np.resize(state[4], len(free)), 150, tokens)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for name, x in zip(("lengths", "held", "count", "granted", "offsets", "positions", "sequences", "slots"), want):
                assert np.array_equal(getattr(got, name).cpu().numpy(), x), (name, seed)
            assert np.array_equal(args[0].cpu().numpy(), want[8]) and np.array_equal(args[4].cpu().numpy(), want[9])


def test_refusals(gpu):
    table, one, free = dev([[0, 1]]), dev([1]), dev([2, 3])
    good = dict(page_rows=16, page_table=table, lengths=one, held=one, new=one, free=free, count=one, tokens=1)
    KV.plan(**good)
    for change in (dict(page_rows=12), dict(page_rows=0), dict(page_rows=1 << 17), dict(tokens=-1), dict(tokens=2**31),
                   dict(page_table=table.long()), dict(page_table=table[0]), dict(lengths=dev([1, 2])), dict(held=one[0]),
                   dict(new=one.cpu()), dict(lengths=one.cpu()), dict(free=free.float()), dict(free=dev([1, 2, 3, 4])[::2]),
                   dict(count=dev([1, 2]))):
        with pytest.raises(ValueError):
            KV.plan(**{**good, **change})
            pytest.fail(f"{change} was not refused")
