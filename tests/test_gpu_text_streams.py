"""A plan or a cache that is dropped while another stream than its own still runs calls with it:
its memory is not given to other tensors before they end."""
import pytest

torch = pytest.importorskip("torch")

from mold_amd import GgmlDType
from mold_amd import text_attention as TA

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _busy():
    """Some tenths of a second of products on the current stream."""
    x = torch.randn((8192, 8192), device="cuda") * 0.01
    for _ in range(20):
        x = x @ x
    return x


def _dropped_on(side, use, own):
    """use() behind other work on `side`, then own()'s memory dropped and everything of its size
    asked for anew; -> use()'s result, and whether the memory came back while side was at work."""
    with torch.cuda.stream(side):
        hold = _busy()
        out = use()
    ptr, size = own()
    others = [torch.full((size,), 255, dtype=torch.uint8, device="cuda") for _ in range(8)]
    early = any(t.data_ptr() <= ptr < t.data_ptr() + size for t in others)
    assert not side.query(), "the other stream has ended too soon for this test"
    torch.cuda.synchronize()
    del hold
    return out, early


def test_a_plan():
    q, k, v = (torch.randn((700, 4, 128), device="cuda").to(BF) for _ in range(3))
    plan = TA.PromptPlan([300, 400], 4, 4, 128)
    want = TA.prompt_attention(q, k, v, plan)
    torch.cuda.synchronize()

    def own():
        nonlocal plan
        at = plan.tiles.data_ptr(), plan.tiles.numel() * 4
        plan = None
        return at
    out, early = _dropped_on(torch.cuda.Stream(), lambda: TA.prompt_attention(q, k, v, plan), own)
    assert not early and torch.equal(out, want)


def test_a_cache():
    cache = TA.KvCache(8, 2, 64, page_tokens=32, dtype=GgmlDType.Q8_0)
    k, v = torch.randn((2, 256, 2, 64), device="cuda")
    slots = torch.arange(256, device="cuda")
    cache.append(k, v, slots)
    q = torch.randn((1, 4, 64), device="cuda").to(BF)
    table, n = torch.arange(8, device="cuda", dtype=torch.int32)[None], torch.tensor([250], dtype=torch.int32, device="cuda")
    want = cache.attend(q, table, n)
    torch.cuda.synchronize()

    def own():
        nonlocal cache
        at = cache.data.data_ptr(), cache.data.numel()
        cache = None
        return at
    out, early = _dropped_on(torch.cuda.Stream(), lambda: cache.attend(q, table, n), own)
    assert not early and torch.equal(out, want)
