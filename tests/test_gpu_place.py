"""Page tables, slots and positions made on the GPU (KvCache.place, KvCache.extend) against the
rules written out on the host; all of it whole numbers, compared as such."""
import ctypes
import random

import pytest

torch = pytest.importorskip("torch")

from mold_amd import GgmlDType, _lib
from mold_amd import text_attention as TA

gpu = pytest.mark.gpu
INT32_MAX = (1 << 31) - 1


def _cache(pages, page=32):
    return TA.KvCache(pages, 1, 64, page_tokens=page, dtype=GgmlDType.Q4_0)


def _place(counts, tokens, width, room, beams, order, page):
    """Every output as lists, by the rules of mq_cache_place."""
    taken = iter(order)
    table, slots, positions, lengths, last, start = [], [], [], [], [], 0
    for count in counts:
        count = max(count, 0)
        columns = min(-(-(count + room) // page), width)
        shared = min(count // page, columns) if beams > 1 else 0
        common = [next(taken, -1) for _ in range(shared)]
        rows = [common + [next(taken, -1) for _ in range(columns - shared)] + [-1] * (width - columns) for _ in range(beams)]
        table += rows
        for p in range(min(count, tokens - len(slots))):
            at = rows[0][p // page] if p // page < width else -1
            slots.append(-1 if at < 0 else at * page + p % page)
            positions.append(p)
        last.append(start + count - 1 if count and start + count <= tokens else -1)
        start += count
        lengths += [count] * beams
    pad = tokens - len(slots)
    return table, slots + [-1] * pad, positions + [0] * pad, lengths, last


def _same(got, want):
    for name, g, w in zip(("table", "slots", "positions", "lengths", "last"), got, want):
        assert g.tolist() == w, name


@gpu
@pytest.mark.parametrize("beams", [1, 2, 5, 64])
@pytest.mark.parametrize("page", [32, 96, 256])
def test_prompts(beams, page):
    """Lengths from none and one to several pages, more sequences than a window's, rows past the last."""
    rng = random.Random(beams * page)
    for n, longest, room in [(1, 1, 0), (1, 1000, 7), (3, page, 0), (24, 1000, 129), (65, 3 * page + 1, page), (1030, 40, 1), (2100, 5, 0)]:
        if n * beams > 12000:
            continue
        counts = [rng.choice([0, 1, page - 1, page, page + 1, longest, rng.randint(0, longest)]) if n > 1 else longest for _ in range(n)]
        counts = [min(c, longest) for c in counts]
        width = max(-(-(c + room) // page) for c in counts) + rng.randint(0, 2)
        need = sum((c // page if beams > 1 else 0) + beams * (-(-(c + room) // page) - (c // page if beams > 1 else 0)) for c in counts)
        cache = _cache(need + 3, page)
        order = list(range(need + 3))
        rng.shuffle(order)
        for tokens in (sum(counts), sum(counts) + 1500):
            c = torch.tensor(counts, dtype=torch.int32, device="cuda")
            _same(cache.place(c, tokens, width, room, beams, torch.tensor(order, dtype=torch.int32, device="cuda")),
                  _place(counts, tokens, width, room, beams, order, page))
        _same(cache.place(c, sum(counts), width, room, beams), _place(counts, sum(counts), width, room, beams, list(range(need + 3)), page))


@gpu
def test_more_sequences_than_16_bits():
    rng = random.Random(3)
    counts = [rng.choice([0, 1, 2, 33]) for _ in range(70001)]
    c = torch.tensor(counts, dtype=torch.int32, device="cuda")
    cache, tokens = _cache(150000), sum(counts) + 3
    at = cache.place(c, tokens, 2)
    _same(at, _place(counts, tokens, 2, 0, 1, range(150000), 32))
    slots, positions, lengths = cache.extend(at.table, at.lengths)
    table = at.table.tolist()
    want = [t[n // 32] if n // 32 < 2 else -1 for t, n in zip(table, counts)]
    assert slots.tolist() == [-1 if p < 0 else 32 * p + n % 32 for p, n in zip(want, counts)]
    assert positions.tolist() == counts and lengths.tolist() == [n + 1 for n in counts]


@gpu
def test_what_does_not_fit():
    """Pages that run out or are not the cache's, a narrow table, rows cut off, counts that mean nothing."""
    page, counts = 32, [70, 0, -5, 33, 200, 1]
    c = torch.tensor(counts, dtype=torch.int32, device="cuda")
    cache = _cache(20)
    for order in ([4, 9], [], [1, -1, 40, 3, 2, 20, 19, 5], list(range(20))):
        valid = [p if 0 <= p < 20 else -1 for p in order]
        for width in (0, 1, 3, 8):
            for tokens in (0, 1, 100, 304, 400):
                got = cache.place(c, tokens, width, 3, 2, torch.tensor(order, dtype=torch.int32, device="cuda"))
                _same(got, _place(counts, tokens, width, 3, 2, valid, page))
    # counts and room at the ends of 32 bits: sums that would wrap
    big = torch.tensor([INT32_MAX, INT32_MAX, -INT32_MAX - 1, INT32_MAX, 3], dtype=torch.int32, device="cuda")
    got = cache.place(big, 50, 4, INT32_MAX, 64)
    want = _place([INT32_MAX], 50, 4, INT32_MAX, 64, range(20), page)
    assert got.table[:64].tolist() == want[0] and got.slots.tolist() == want[1] and got.positions.tolist() == want[2]
    assert (got.table[64:].reshape(-1) >= -1).all() and got.last.tolist() == [-1] * 5
    assert got.lengths.view(5, 64)[:, 0].tolist() == [INT32_MAX, INT32_MAX, 0, INT32_MAX, 3]


@gpu
def test_no_sequences_and_no_pages():
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    got = _cache(4).place(none, 3, 2)
    assert got.table.shape == (0, 2) and got.slots.tolist() == [-1] * 3 and got.positions.tolist() == [0] * 3 and got.last.shape == (0,)
    got = _cache(0).place(torch.tensor([3, 1], dtype=torch.int32, device="cuda"), 4, 1)
    assert got.table.tolist() == [[-1], [-1]] and got.slots.tolist() == [-1] * 4 and got.last.tolist() == [2, 3]
    slots, positions, lengths = _cache(4).extend(torch.empty((0, 3), dtype=torch.int32, device="cuda"), none)
    assert slots.shape == positions.shape == lengths.shape == (0,)


def _extend(table, held, counts, tokens, page, pages):
    width, slots, positions = len(table[0]) if table else 0, [], []
    for row, h, c in zip(table, held, counts):
        for p in range(h, h + max(c, 0)):
            if len(slots) == tokens:
                break
            at = row[p // page] if 0 <= p // page < width else -1
            slots.append(at * page + p % page if 0 <= at < pages else -1)
            positions.append(p)
    pad = tokens - len(slots)
    return slots + [-1] * pad, positions + [0] * pad, [min(h + max(c, 0), INT32_MAX) for h, c in zip(held, counts)]


@gpu
def test_sequences_that_go_on():
    rng = random.Random(3)
    for n, width, page in [(1, 1, 32), (7, 3, 96), (200, 40, 64), (1500, 4, 32)]:
        pages = 50
        cache = _cache(pages, page)
        table = [[rng.choice([-1, pages, INT32_MAX] + list(range(pages)) * 5) for _ in range(width)] for _ in range(n)]
        held = [rng.choice([0, width * page - 1, width * page, width * page + 5, -3, INT32_MAX - 1, rng.randint(0, width * page)]) for _ in range(n)]
        t, h = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (table, held))
        want = _extend(table, held, [1] * n, n, page, pages)
        for got in (cache.extend(t, h), cache.extend(t, h, torch.ones_like(h), n), cache.extend(torch.cat([t, t], 1)[:, :width], h),
                    cache.extend(t.t().contiguous().t(), torch.stack([h, h], 1)[:, 1])):
            assert [x.tolist() for x in got] == list(want)
        counts = [rng.choice([0, 1, 2, page, -1, 2 * page + 1]) for _ in range(n)]
        c, total = torch.tensor(counts, dtype=torch.int32, device="cuda"), sum(max(x, 0) for x in counts)
        for tokens in (total, total + 3, max(total - 5, 0)):
            assert [x.tolist() for x in cache.extend(t, h, c, tokens)] == list(_extend(table, held, counts, tokens, page, pages)), (n, tokens)
        assert h.tolist() == held and t.tolist() == table
    empty = torch.empty((3, 0), dtype=torch.int32, device="cuda")
    slots, positions, lengths = _cache(4).extend(empty, torch.tensor([0, 5, 9], dtype=torch.int32, device="cuda"))
    assert slots.tolist() == [-1] * 3 and positions.tolist() == [0, 5, 9] and lengths.tolist() == [1, 6, 10]


@gpu
def test_the_slots_are_those_of_the_table():
    """place, then extend token by token, name the slots that KvCache.slots finds in the table."""
    cache = _cache(100, 32)
    at = cache.place(torch.tensor([40, 3, 64], dtype=torch.int32, device="cuda"), 107, 5, room=70, beams=3)
    pos = at.positions.view(1, -1).expand(9, -1).contiguous()
    every = cache.slots(at.table, pos)
    seq = torch.repeat_interleave(torch.arange(3, device="cuda"), torch.tensor([40, 3, 64], device="cuda"))
    assert torch.equal(at.slots, every[3 * seq, torch.arange(107, device="cuda")])
    lengths = at.lengths
    seen = set(at.slots.tolist())
    for _ in range(70):
        slots, positions, after = cache.extend(at.table, lengths)
        assert torch.equal(positions, lengths.long()) and torch.equal(after, lengths + 1)
        assert torch.equal(slots, cache.slots(at.table, positions[:, None])[:, 0])
        lengths = after
        seen.update(slots.view(3, 3)[:, 1:].reshape(-1).tolist())
    assert len(seen) == 107 + 6 * 70 and -1 not in seen      # every beam writes to slots of its own


@gpu
def test_captured():
    cache = _cache(400, 32)
    counts = torch.tensor([5, 40, 0, 99], dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        cache.place(counts, 300, 6, room=9, beams=2)
        with torch.cuda.graph(graph, stream=s):
            placed = cache.place(counts, 300, 6, room=9, beams=2)
            more = cache.extend(placed.table, placed.lengths)
    torch.cuda.current_stream().wait_stream(s)
    for values in ([5, 40, 0, 99], [0, 0, 0, 1], [150, 1, 150, 3], [32, 64, 96, 128]):
        counts.copy_(torch.tensor(values, dtype=torch.int32))
        want = cache.place(counts, 300, 6, room=9, beams=2)
        after = cache.extend(want.table, want.lengths)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((*placed, *more), (*want, *after))), values


@gpu
def test_refusals():
    cache = _cache(4)
    c = torch.tensor([1, 2], dtype=torch.int32, device="cuda")
    t = torch.zeros((2, 3), dtype=torch.int32, device="cuda")
    for call in (lambda: cache.place(c.long(), 3, 1), lambda: cache.place(c[None], 3, 1), lambda: cache.place(c.cpu(), 3, 1), lambda: cache.place(c, -1, 1),
                 lambda: cache.place(c, 3, -1), lambda: cache.place(c, 3, 1, beams=0), lambda: cache.place(c, 3, 1, pages=c.long()),
                 lambda: cache.extend(t, c.long()), lambda: cache.extend(t[:1], c), lambda: cache.extend(t.long(), c), lambda: cache.extend(t, c, c),
                 lambda: cache.extend(t, c, c[:1], 3), lambda: cache.extend(t, c, tokens=-1), lambda: cache.extend(t.cpu(), c)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: cache.place(c, 3, 1, room=-1), lambda: cache.place(c, 3, 1, room=1 << 31), lambda: cache.place(c, 3, 1, beams=65)):
        with pytest.raises((ValueError, RuntimeError)):
            call()


def test_refusals_of_the_library():
    """On the CPU: every fault is found before anything is launched."""
    lib, a, bad = _lib.load(), 4096, _lib.MQ_E_INVALID
    cache = _lib.KvCacheC(a, 4, 8, 2, 128, 64)
    place = dict(counts=a, n=3, beams=2, room=1, pages=a, page_count=4, table=a, stride=5, width=5, tokens=7, slots=a, positions=a, lengths=a, last=a, stream=None)
    for change in (dict(counts=None), dict(n=-1), dict(n=(1 << 20) + 1), dict(beams=0), dict(beams=65), dict(room=-1), dict(room=1 << 31), dict(page_count=-1),
                   dict(page_count=1 << 31), dict(table=None), dict(stride=4), dict(stride=1 << 40), dict(width=-1), dict(width=1 << 31, stride=1 << 31), dict(tokens=-1), dict(tokens=1 << 31),
                   dict(slots=None), dict(positions=None), dict(lengths=None), dict(last=None), dict(slots=a + 4), dict(counts=a + 2), dict(table=a + 1),
                   dict(last=a + 4), dict(positions=a + 4), dict(lengths=a + 2), dict(pages=a + 2)):
        assert lib.mq_cache_place(ctypes.byref(cache), *{**place, **change}.values()) == bad, change
    assert lib.mq_cache_place(ctypes.byref(cache), *{**place, "n": 0, "tokens": 0}.values()) == 0
    extend = dict(held=a, counts=a, n=3, table=a, stride=5, width=5, tokens=7, slots=a, positions=a, lengths=a, stream=None)
    for change in (dict(held=None), dict(n=-1), dict(n=(1 << 20) + 1), dict(table=None), dict(stride=4), dict(width=-1), dict(tokens=-1), dict(slots=None),
                   dict(positions=None), dict(lengths=None), dict(held=a + 2), dict(counts=a + 1), dict(slots=a + 4)):
        assert lib.mq_cache_extend(ctypes.byref(cache), *{**extend, **change}.values()) == bad, change
    cache.page_tokens = 48
    assert lib.mq_cache_place(ctypes.byref(cache), *place.values()) == bad and lib.mq_cache_extend(ctypes.byref(cache), *extend.values()) == bad
    assert lib.mq_cache_place(None, *place.values()) == bad and lib.mq_cache_extend(None, *extend.values()) == bad
