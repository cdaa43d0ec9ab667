"""What the text attention's entry points take and refuse: calls that something records, tensors
that start off 16 bytes, an output that autograd watches, one token's strides."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from mold_amd import GgmlDType, _lib
from mold_amd import text_attention as TA

gpu = pytest.mark.gpu
BF = torch.bfloat16


def _cache(dtype=GgmlDType.BF16, tokens=40):
    cache = TA.KvCache(2, 2, 64, page_tokens=32, dtype=dtype)
    g = torch.Generator(device="cuda").manual_seed(5)
    k, v = torch.randn((2, tokens, 2, 64), device="cuda", generator=g)
    slots = torch.arange(tokens, device="cuda")
    cache.append(k, v, slots)
    return cache, slots


def _off(t):
    """t's values in a contiguous tensor that starts one element off 16 bytes."""
    off = torch.empty(t.numel() + 8, dtype=t.dtype, device=t.device)[1:t.numel() + 1].view(t.shape)
    assert off.is_contiguous() and off.data_ptr() % 16
    return off.copy_(t)


@gpu
def test_a_read_that_is_recorded_is_refused():
    """A trace would keep the allocations and not the kernel: its replay would return memory as it is."""
    cache, slots = _cache()
    with pytest.raises(ValueError):
        torch.jit.trace(lambda s: cache.read(s), (slots,), check_trace=False)
    with torch.autograd.forward_ad.dual_level(), pytest.raises(ValueError):
        cache.read(slots)
    assert cache.read(slots)[0].shape == (40, 2, 64)


@gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_prompts_off_16_bytes(dim):
    g = torch.Generator(device="cuda").manual_seed(1)
    for n, heads, kv in ((50, 4, 2), (1, 1, 1)):
        plan = TA.PromptPlan([n], heads, kv, dim)
        q, k, v = (torch.randn((n, h, dim), device="cuda", generator=g).to(BF) for h in (heads, kv, kv))
        want = TA.prompt_attention(q, k, v, plan)
        for off in ((_off(q), k, v), (q, _off(k), v), (q, k, _off(v)), (_off(q), _off(k), _off(v))):
            assert torch.equal(TA.prompt_attention(*off, plan), want), n
        wide = torch.nn.functional.pad(q, (1, 7))[..., 1:dim + 1]     # of one token and head: contiguous too
        assert torch.equal(TA.prompt_attention(wide, k, v, plan), want), n


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, BF], ids=["f32", "bf16"])
def test_cache_calls_off_16_bytes(dtype):
    g = torch.Generator(device="cuda").manual_seed(2)
    slots = torch.arange(40, device="cuda")
    k, v = torch.randn((2, 40, 2, 64), device="cuda", generator=g).to(dtype)
    caches = [TA.KvCache(2, 2, 64, page_tokens=32, dtype=GgmlDType.Q8_0) for _ in range(4)]
    for c, (a, b) in zip(caches, ((k, v), (_off(k), v), (k, _off(v)), (_off(k), _off(v)))):
        c.append(a, b, slots)
        assert all(torch.equal(x, y) for x, y in zip(c.read(slots), caches[0].read(slots)))
    q = torch.randn((1, 4, 64), device="cuda", generator=g).to(BF)
    table, n = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"), torch.tensor([40], dtype=torch.int32, device="cuda")
    assert torch.equal(caches[0].attend(_off(q), table, n), caches[0].attend(q, table, n))


@gpu
def test_an_out_that_requires_gradients_is_refused():
    """As any write in place into it; without gradient recording it is written."""
    q, k, v = (torch.randn((8, 2, 64), device="cuda").to(BF) for _ in range(3))
    plan = TA.PromptPlan([8], 2, 2, 64)
    cache, _ = _cache()
    table = torch.tensor([[0, 1]] * 8, dtype=torch.int32, device="cuda")
    n = torch.arange(8, dtype=torch.int32, device="cuda")
    for call in (lambda **kw: TA.prompt_attention(q, k, v, plan, **kw), lambda **kw: cache.attend(q, table, n, **kw)):
        out = torch.zeros((8, 2, 64), device="cuda", dtype=BF, requires_grad=True)
        for given in (out, out[:], (out * 1)):
            with pytest.raises(ValueError):
                call(out=given)
        assert not out.detach().any()
        with torch.no_grad():
            assert call(out=out) is out
        assert torch.equal(out.detach(), call())


@gpu
def test_one_token_has_any_token_stride():
    """A single row is not apart from another one: its token stride may be anything, 0 too."""
    lib, plan, n = _lib.load(), _lib.PromptPlanC(), (ctypes.c_int64 * 1)(1)
    for heads in (1, 4):
        q, k, v = (torch.randn((1, heads, 64), device="cuda").to(BF) for _ in range(3))
        tiles = TA.PromptPlan([1], heads, heads, 64)
        assert lib.mq_prompt_plan_make(n, 1, heads, heads, 64, ctypes.byref(plan), None, 0) == 0
        for stride in (0, 8, 64 * heads, 1 << 20):
            out = torch.zeros_like(q)
            args = [x for t in (q, k, v) for x in (t.data_ptr(), stride, 64)]
            assert lib.mq_prompt_attention(ctypes.byref(plan), tiles.tiles.data_ptr(), *args, 0.125, out.data_ptr(), stride, 64,
                                           torch.cuda.current_stream().cuda_stream) == 0, (heads, stride)
            assert torch.equal(out, v), (heads, stride)
