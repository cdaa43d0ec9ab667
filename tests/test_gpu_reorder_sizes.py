"""BeamStates.reorder over long sequences: the page table's columns are shared by several workgroups."""
import random

import pytest

torch = pytest.importorskip("torch")

from mold_amd import GgmlDType
from mold_amd.beams import BeamStates
from tests.test_gpu_beams import _raw, _states
from tests.test_gpu_place_sizes import _i32, _least

pytestmark = pytest.mark.gpu


def _tokens(cache, pages, tail):
    """The bits of the first `tail` tokens of each of `pages`, as they are read."""
    slots = (pages.reshape(-1, 1).long() * cache.page_tokens + torch.arange(tail)).reshape(-1)
    return torch.stack(cache.read(slots.cuda())).view(torch.int16).cpu()


@pytest.mark.parametrize("n,beams,full,tail", [(1, 2, 63, 1), (1, 5, 64, 0), (2, 64, 65, 31), (3, 3, 128, 32), (7, 4, 129, 5), (1, 64, 5000, 40), (30, 2, 700, 9), (2100, 2, 130, 3)])
def test_long_tables(n, beams, full, tail):
    """Whole pages of any numbers, which the kernel only moves about; partial ones of the cache's."""
    rng, page = random.Random(full), 64
    width, g = full + 2, torch.Generator().manual_seed(full)
    table = torch.randint(0, 1 << 30, (n, beams, width), dtype=torch.int32, generator=g)
    order = torch.randperm(n * beams * 2, generator=g).to(torch.int32)
    table[:, :, full:] = order.view(n, beams, 2)
    cache = _states(1, n * beams * 2, 1, 64, page, GgmlDType.Q4_0)[0]
    parents = torch.randint(-1, beams + 1, (n, beams), dtype=torch.int32, generator=g)
    parents[rng.randrange(n)] = torch.arange(beams)          # of one request every beam goes on as it is
    whose = torch.where((parents < 0) | (parents >= beams), torch.arange(beams), parents).long()
    length = full * page + tail
    raw, held = _raw(cache), _tokens(cache, torch.gather(table, 1, whose[:, :, None].expand(n, beams, width))[:, :, full], tail)
    dev = table.view(n * beams, width).cuda()
    BeamStates([cache]).reorder(dev, _i32([length] * n * beams), parents.cuda())
    got = dev.cpu().view(n, beams, width)
    want = torch.gather(table, 1, whose[:, :, None].expand(n, beams, width))
    assert torch.equal(got[:, :, :full], want[:, :, :full]) and torch.equal(got[:, :, full + 1], table[:, :, full + 1])
    if not tail:
        assert torch.equal(got[:, :, full], table[:, :, full]) and torch.equal(_raw(cache), raw)
        return
    assert torch.equal(got[:, :, full].sort(1).values, table[:, :, full].sort(1).values)
    assert torch.equal(_tokens(cache, got[:, :, full], tail), held)


def test_its_time_is_that_of_the_table():
    """4 requests of 64 beams over 31 250 whole pages, and torch's gather of the same rows: the same bytes."""
    n, beams, full, page = 4, 64, 31250, 32
    cache = _states(1, n * beams * 2, 1, 64, page, GgmlDType.Q4_0)[0]
    table = torch.zeros((n * beams, full + 2), dtype=torch.int32, device="cuda")
    table[:, full:] = torch.arange(n * beams * 2, device="cuda").view(-1, 2)
    lengths, states = _i32([full * page + 7] * n * beams), BeamStates([cache])
    parents = _i32([[max(j - 1, 0) for j in range(beams)]] * n)
    rows = (torch.arange(n, device="cuda")[:, None] * beams + parents).view(-1)
    ours, plain = _least(lambda: states.reorder(table, lengths, parents)), _least(lambda: table.copy_(table[rows]))
    assert ours <= 8 * plain, (ours, plain)


@pytest.mark.parametrize("caches", [255, 256])
def test_as_many_caches_as_one_reordering_takes(caches):
    """Each by itself: its copies are of its own bytes."""
    page, length = 32, 21
    alike = _states(caches, 8, 1, 64, page, GgmlDType.Q4_0)
    pages = torch.tensor([2, 2, 4, 4])       # the parents'
    held = [_tokens(c, pages, length) for c in alike]
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(4, 2)
    BeamStates(alike).reorder(table, _i32([length] * 4), _i32([[1, 1], [0, 0]]))
    assert table.tolist() == [[0, 1], [2, 3], [4, 5], [6, 7]]
    assert all(torch.equal(_tokens(c, torch.tensor([0, 2, 4, 6]), length), h) for c, h in zip(alike, held))
    with pytest.raises(ValueError, match="256"):
        BeamStates(alike + _states(257 - caches, 8, 1, 64, page, GgmlDType.Q4_0))
