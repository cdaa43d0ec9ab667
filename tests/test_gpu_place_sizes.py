"""KvCache.place at sizes where its work is more than a launch: results against the rules, and times that
grow with the work.

A time is the least of several, compared with that of other calls of the same operator, with
room for a factor of four or more beyond what the work gives."""
import random

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from tests.test_gpu_place import INT32_MAX, _cache, _extend, _place, _same

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _least(call, times=5):
    call()
    spent = []
    for _ in range(times):
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        start.record()
        call()
        end.record()
        torch.cuda.synchronize()
        spent.append(start.elapsed_time(end))
    return min(spent)


@pytest.mark.parametrize("n,beams,longest,page", [(1, 64, 5000, 32), (3, 64, 900, 32), (5, 7, 40000, 32), (4, 2, 131072, 32), (9, 64, 2000, 64), (2, 1, 300000, 32)])
def test_wide_tables(n, beams, longest, page):
    """Rows of a few sequences that several workgroups write, whole ones and parts."""
    rng = random.Random(n * beams)
    counts = [longest] + [rng.choice([0, 1, page, longest // 2, rng.randint(0, longest)]) for _ in range(n - 1)]
    room, width = 70, -(-(longest + 70) // page) + 1
    need = sum((c // page if beams > 1 else 0) + beams * (-(-(c + room) // page) - (c // page if beams > 1 else 0)) for c in counts)
    cache, order = _cache(need, page), list(range(need))
    rng.shuffle(order)
    tokens = sum(counts) + 5
    _same(cache.place(_i32(counts), tokens, width, room, beams, _i32(order)), _place(counts, tokens, width, room, beams, order, page))


def test_a_few_wide_rows_take_what_many_narrow_ones_do():
    """512 000 table entries of 4 prompts with 64 beams, and of 256 with four."""
    wide, narrow = _cache(60000, 64), _cache(600000, 64)
    few, many = _i32([127900] * 4), _i32([2000] * 256)
    one = _least(lambda: wide.place(few, 10, 2004, 256, 64))
    other = _least(lambda: narrow.place(many, 10, 501, 30000, 4))
    assert one <= 4 * other, (one, other)


@pytest.mark.parametrize("n", [4095, 4096, 4097, 5121, 8192, 20003])
@pytest.mark.parametrize("beams", [1, 2, 7])
def test_many_sequences(n, beams):
    """On both sides of where the sequences' sums are taken beforehand; windows of nothing but empty sequences."""
    rng = random.Random(n + beams)
    counts = [rng.choice([0, 0, 1, 2, 33]) for _ in range(n)]
    counts[1000:3500] = [0] * 2500
    counts[-1] = 40
    page, room, width = 32, 3, 2
    need = sum((c // page if beams > 1 else 0) + beams * (-(-(c + room) // page) - (c // page if beams > 1 else 0)) for c in counts)
    cache, c = _cache(need, page), _i32(counts)
    for tokens in (sum(counts), sum(counts) + 3000, sum(counts) // 2 + 1):
        _same(cache.place(c, tokens, width, room, beams), _place(counts, tokens, width, room, beams, range(need), page))


@pytest.mark.parametrize("n", [4096, 4097, 6000, 30000])
def test_many_sequences_that_go_on(n):
    rng = random.Random(n)
    cache, width = _cache(50, 32), 2
    table = [[rng.choice([-1, 50, rng.randrange(50)]) for _ in range(width)] for _ in range(n)]
    held = [rng.choice([0, 63, 64, -3, INT32_MAX - 1, rng.randint(0, 64)]) for _ in range(n)]
    counts = [rng.choice([0, 0, 1, 2, 33, -1]) for _ in range(n)]
    counts[1000:3500] = [0] * 2500
    total = sum(max(c, 0) for c in counts)
    t, h, c = _i32(table), _i32(held), _i32(counts)
    for tokens in (total, total + 2000, total // 3):
        assert [x.tolist() for x in cache.extend(t, h, c, tokens)] == list(_extend(table, held, counts, tokens, 32, 50)), tokens
    assert h.tolist() == held and c.tolist() == counts and t.tolist() == table


def test_as_many_as_there_can_be():
    """2^20 sequences, their sums past 2^31 at the end."""
    n, beams, page = 1 << 20, 3, 32
    counts = np.random.default_rng(1).integers(0, 70, n)
    big = counts.copy()
    big[-2000:] = INT32_MAX
    columns, shared = -(-(counts + 5) // page), counts // page
    need = shared + beams * (columns - shared)
    first, start = np.cumsum(need) - need, np.cumsum(counts) - counts
    at = _cache(1).place(_i32(big), 1 << 22, 3, 5, beams)          # one page: whoever comes first
    keep = n - 2000
    pages = at.table.cpu().numpy()
    assert (pages <= 0).all() and (pages == 0).sum() == (beams if shared[np.nonzero(need)[0][0]] else 1)
    assert np.array_equal(at.lengths.cpu().numpy().reshape(n, beams), np.repeat(big[:, None], beams, 1))
    got = at.positions.cpu().numpy()
    seq = np.searchsorted(start, np.arange(1 << 22), side="right") - 1
    assert np.array_equal(got, np.arange(1 << 22) - start[seq])
    last = np.where((counts > 0) & (start + counts <= 1 << 22), start + counts - 1, -1)
    assert np.array_equal(at.last.cpu().numpy()[:keep], last[:keep]) and (at.last[keep:] == -1).all()
    cache = _cache(int(need.sum()), page)
    at = cache.place(_i32(counts), int(counts.sum()), 3, 5, beams)
    c, j = np.arange(3)[None, None], np.arange(beams)[None, :, None]
    sh, co = shared[:, None, None], columns[:, None, None]
    want = np.where(c < co, first[:, None, None] + np.where(c < sh, c, sh + j * (co - sh) + c - sh), -1)
    assert np.array_equal(at.table.cpu().numpy(), want.reshape(n * beams, 3))
    seq = np.repeat(np.arange(n), counts)
    pos = np.arange(counts.sum()) - start[seq]
    assert np.array_equal(at.positions.cpu().numpy(), pos)
    assert np.array_equal(at.slots.cpu().numpy(), want[seq, 0, pos // page] * page + pos % page)


def test_times_grow_with_the_sequences():
    """64 times as many take no more than 64 times as long."""
    few, many = 1 << 14, 1 << 20
    cache, one = _cache(many, 32), {n: torch.ones(n, dtype=torch.int32, device="cuda") for n in (few, many)}
    table = {n: torch.zeros((n, 1), dtype=torch.int32, device="cuda") for n in one}
    for call in (lambda n: cache.place(one[n], n, 1, 10), lambda n: cache.extend(table[n], one[n], one[n], n)):
        small, large = _least(lambda: call(few)), _least(lambda: call(many))
        assert large <= 64 * small, (small, large)


def test_many_sequences_captured():
    """The launches of one call, replayed."""
    n = 9000
    cache, counts = _cache(3 * n, 32), torch.zeros(n, dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        cache.place(counts, 4 * n, 3, 1, 2)
        with torch.cuda.graph(graph, stream=s):
            placed = cache.place(counts, 4 * n, 3, 1, 2)
            more = cache.extend(placed.table[::2], placed.lengths[::2].contiguous(), counts, 4 * n)
    torch.cuda.current_stream().wait_stream(s)
    for seed in range(4):
        counts.copy_(torch.randint(0, 70 >> seed, (n,), generator=torch.Generator().manual_seed(seed)))
        want = cache.place(counts, 4 * n, 3, 1, 2)
        after = cache.extend(want.table[::2], want.lengths[::2].contiguous(), counts, 4 * n)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((*placed, *more), (*want, *after))), seed
