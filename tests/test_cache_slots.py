"""KvCache.slots on the CPU (it is torch operations over the page table): positions past a
sequence's table have no slot, as negative ones have none.  On a GPU an index past the table
would be a device assertion, which ends the process."""
from types import SimpleNamespace

import pytest

torch = pytest.importorskip("torch")

from mold_amd.text_attention import KvCache

INT32_MAX = (1 << 31) - 1


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_positions_past_the_table(dtype):
    table = torch.tensor([[4, 1], [0, 5], [-1, 7]], dtype=torch.int32)
    pos = torch.tensor([[0, 63, 64, INT32_MAX], [-1, 33, 1000, 95], [31, 32, 65, -INT32_MAX]], dtype=dtype)
    got = KvCache.slots(SimpleNamespace(page_tokens=32), table, pos)
    assert got.dtype == torch.int64
    assert got[:2].tolist() == [[128, 63, -1, -1], [-1, 161, -1, -1]]
    assert got[2, 0] < 0 and got[2, 1:].tolist() == [224, -1, -1]      # a table's -1 names no page


def test_a_table_without_pages():
    none = torch.empty((2, 0), dtype=torch.int32)
    got = KvCache.slots(SimpleNamespace(page_tokens=32), none, torch.tensor([[0, 5, -3], [1, 2, 3]]))
    assert got.tolist() == [[-1] * 3] * 2
    assert KvCache.slots(SimpleNamespace(page_tokens=32), none[:0], torch.empty((0, 4), dtype=torch.int64)).shape == (0, 4)
