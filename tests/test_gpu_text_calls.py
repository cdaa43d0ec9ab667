"""What the text attention's entry points take and refuse: calls that something records."""
import pytest

torch = pytest.importorskip("torch")

from mold_amd import GgmlDType
from mold_amd import text_attention as TA

gpu = pytest.mark.gpu


def _cache(dtype=GgmlDType.BF16, tokens=40):
    cache = TA.KvCache(2, 2, 64, page_tokens=32, dtype=dtype)
    g = torch.Generator(device="cuda").manual_seed(5)
    k, v = torch.randn((2, tokens, 2, 64), device="cuda", generator=g)
    slots = torch.arange(tokens, device="cuda")
    cache.append(k, v, slots)
    return cache, slots


@gpu
def test_a_read_that_is_recorded_is_refused():
    """A trace would keep the allocations and not the kernel: its replay would return memory as it is."""
    cache, slots = _cache()
    with pytest.raises(ValueError):
        torch.jit.trace(lambda s: cache.read(s), (slots,), check_trace=False)
    with torch.autograd.forward_ad.dual_level(), pytest.raises(ValueError):
        cache.read(slots)
    assert cache.read(slots)[0].shape == (40, 2, 64)
