"""Assembly checks of the launches around place_kernel (CPU; needs hipcc, skipped without it): no private
array in scratch memory."""
from tests.test_build_checks import _asm, _functions, pytestmark  # noqa: F401


def test_sums_and_lengths_keep_to_registers(tmp_path):
    funcs = {k: v for k, v in _functions(_asm(tmp_path, "mq_place.hip")).items() if "ScratchSize" in v[1]}
    assert sorted(name for k in funcs for name in ("place_kernel", "put_lengths", "sum_windows") if name in k) == ["place_kernel", "put_lengths", "sum_windows"]
    assert len(funcs) == 3 and all(meta["ScratchSize"] == 0 for _, meta in funcs.values())
