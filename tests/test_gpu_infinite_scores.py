"""Keys whose scores are minus infinity, whole runs of 32 of them and before a row's first finite
one, in mq_prompt_attention and mq_cache_attention at scales below and above 1 / log2(e) = 0.693:
by the definition they weigh nothing beside a finite score, and a row that sees nothing else
has no value (0 / 0).

Against float64; the bound is that of the finite cases (2.4e-3 from the roundings of
probabilities and output to bf16, 3e-3 asserted over the rows that have a value)."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from mold_amd import GgmlDType, _lib
from mold_amd import text_attention as TA
from tests.test_gpu_decode_attention import _Batch
from tests.test_gpu_prompt_attention import _inputs, _ref, _run, _run_whole

gpu = pytest.mark.gpu
BOUND = 3e-3
SCALES = [0.5, 0.69, 0.7, 1.0, 30.0]
RUNS = [[(0, 32)], [(32, 64)], [(0, 64)], [(0, 128)], [(0, 96), (128, 160)], [(32, 33), (64, 96)]]


def _check(out, ref, what):
    out = out.double().cpu()
    assert torch.equal(torch.isnan(out), torch.isnan(ref)), what
    ok = ~torch.isnan(ref)
    assert ((out - ref)[ok].norm() / ref[ok].norm()).item() < BOUND, what


@gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("scale", SCALES)
def test_prompts(dim, scale):
    lengths = [200, 45]
    for heads, kv in ((4, 1), (6, 2), (1, 1)):
        q, k, v = (t.contiguous() for t in _inputs(lengths, heads, kv, dim, sharp=0.2 / max(1.0, scale)))
        q[..., 0] = q[..., 0].abs() + 0.01
        for runs in RUNS:
            bad = k.clone()
            for a, b in runs:
                bad[a:b, :, 0] = float("-inf")
            ref = _ref(q, bad, v, lengths, scale=scale)
            assert torch.isnan(ref).any() == (runs[0][0] == 0)
            _check(_run(q, bad, v, lengths, scale=scale), ref, (heads, runs, "split"))
    whole = _run_whole(q, bad, v, lengths)               # at the default scale, for its asserted form
    _check(whole, _ref(q, bad, v, lengths), "whole")


@gpu
@pytest.mark.parametrize("scale", SCALES)
def test_prompts_in_whole_tiles(scale):
    """So many tiles that none is split over the keys."""
    lengths = [200] + [1] * 2000
    q, k, v = (t.contiguous() for t in _inputs(lengths, 4, 2, 128, sharp=0.2 / max(1.0, scale)))
    plan = TA.PromptPlan(lengths, 4, 2, 128)
    assert plan.c.parts == 1
    q[..., 0] = q[..., 0].abs() + 0.01
    for runs in RUNS:
        bad = k.clone()
        for a, b in runs:
            bad[a:b, :, 0] = float("-inf")
        out = TA.prompt_attention(q, bad, v, plan, scale=scale)
        _check(out[:200], _ref(q[:200], bad[:200], v[:200], [200], scale=scale), runs)


@gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("scale", SCALES)
def test_cache(dim, scale):
    """Tables of up to 32 tiles (a workgroup a sequence and head) and longer ones (runs of the
    whole batch's tiles), with runs of every other tile, so that a wave's first may be one."""
    for lengths in ([33, 64, 200, 32, 1000], [5000, 40, 33, 2500]):
        b = _Batch(lengths, 4, 2, dim, GgmlDType.BF16, sharp=0.2 / max(1.0, scale))
        b.q[..., 0] = b.q[..., 0].abs() + 0.01
        keys = [b.cache.read(s)[0] for s in b.slots]
        values = [b.cache.read(s)[1] for s in b.slots]
        for every in (False, True):
            for slots, k, v in zip(b.slots, keys, values):
                k = k.clone()
                at = torch.arange(len(k), device="cuda") // 32
                k[(at % 2 == 0) if every else (at == 0), :, 0] = float("-inf")
                b.cache.append(k, v, slots)
            ref = b.ref(scale)
            assert torch.isnan(ref).any() == (32 in lengths)
            _check(b.run(scale=scale), ref, (lengths, every))


def test_scales_that_pass_float32_in_bits_are_refused():
    """The kernels work in base 2: scale times log2(e) has to be a float32 too."""
    lib, plan, n = _lib.load(), _lib.PromptPlanC(), (ctypes.c_int64 * 1)(3)
    cache = _lib.KvCacheC(4096, 3, 30, 2, 64, 32)
    assert lib.mq_prompt_plan_make(n, 1, 2, 2, 64, ctypes.byref(plan), None, 0) == 0
    for scale in (2.4e38, 3e38, float("inf"), float("nan"), 0.0, -1.0):
        args = (ctypes.byref(plan), 4096) + (4096, 128, 64) * 3 + (scale, 1 << 20, 128, 64, None)
        assert lib.mq_prompt_attention(*args) == _lib.MQ_E_INVALID, scale
        assert lib.mq_cache_attention(ctypes.byref(cache), 4096, 128, 64, 2, 2, 4096, 2, 2, 4096, scale, 1 << 20, 128, 64, None, 0,
                                      None) == _lib.MQ_E_INVALID, scale
