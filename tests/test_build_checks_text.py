"""Assembly checks of the decoder's step and beam search kernels (CPU; needs hipcc, skipped without it):
rows, keys and candidates stay in registers, no private array in scratch memory."""
import pytest

from tests.test_build_checks import _asm, _functions, pytestmark  # noqa: F401


@pytest.mark.parametrize("src,kernels", [("mq_heads.hip", 4 + 12), ("mq_place.hip", 1), ("mq_beams.hip", 2 * 2 + 1 + 1 + 6), ("mq_cache.hip", 24)])
def test_kernels_keep_to_registers(tmp_path, src, kernels):
    funcs = {k: v for k, v in _functions(_asm(tmp_path, src)).items() if "_kernel" in k and "ScratchSize" in v[1]}
    assert len(funcs) == kernels
    for name, (_, meta) in funcs.items():
        assert meta["ScratchSize"] == 0, (name, meta)
