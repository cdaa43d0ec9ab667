"""BeamStates.reorder changes its page table in place and says so to autograd, as torch's own
in-place operations do."""
import pytest

torch = pytest.importorskip("torch")

from mold_amd import GgmlDType
from mold_amd import text_attention as TA
from mold_amd.beams import BeamStates

pytestmark = pytest.mark.gpu


def _inputs():
    cache = TA.KvCache(8, 1, 64, page_tokens=32, dtype=GgmlDType.Q4_0)
    cache.data.zero_()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    return BeamStates([cache]), i32([[0, 1], [2, 3], [4, 5], [6, 7]]), i32([40] * 4), i32([[1, 1], [0, 1]])


def test_a_table_saved_for_backward_is_missed():
    states, table, lengths, parents = _inputs()
    w = torch.ones((4, 2), device="cuda", requires_grad=True)
    y = (w * table).sum()
    before = table._version
    states.reorder(table, lengths, parents)
    assert table._version > before and table.tolist() == [[2, 1], [2, 3], [4, 5], [6, 7]]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_what_writes_nothing_changes_no_version():
    states, table, lengths, parents = _inputs()
    before = table._version
    states.reorder(table, lengths, parents.view(4, 1))
    states.reorder(table[:0], lengths[:0], parents[:0])
    assert table._version == before


def test_tables_made_under_inference_mode():
    """They have no version: reordered outside of it too, as before."""
    with torch.inference_mode():
        states, table, lengths, parents = _inputs()
        states.reorder(table, lengths, parents)
        assert table.tolist() == [[2, 1], [2, 3], [4, 5], [6, 7]]
    states.reorder(table, lengths, parents)      # the second beam keeps its page, the first takes its own again
    assert table.tolist() == [[2, 1], [2, 3], [4, 5], [6, 7]]
