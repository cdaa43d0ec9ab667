"""KvCache.place at sizes where its work is more than a launch: results against the rules, and times that
grow with the work.

A time is the least of several, compared with that of other calls of the same operator, with
room for a factor of four or more beyond what the work gives."""
import random

import pytest

torch = pytest.importorskip("torch")

from tests.test_gpu_place import _cache, _place, _same

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
