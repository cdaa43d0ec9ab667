"""rotate_heads and KvCache.append_rotated at the most tokens that they document, and past them.

Every token is the same one row of q, k and v at a position that repeats, so that the results of a
few thousand tokens, which test_gpu_rotated_heads compares with float64, are those of all."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from mold_amd import GgmlDType, MoldqError, _lib
from mold_amd import text_attention as TA

gpu = pytest.mark.gpu
PERIOD = 4096


def _inputs(n, dim):
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn((1, 1, dim), device="cuda", generator=g).bfloat16().expand(n, 1, dim) for _ in range(3))
    freq = 1e4 ** (-torch.arange(dim // 2, device="cuda", dtype=torch.float32) / (dim // 2))
    return q, k, v, torch.arange(n, device="cuda") % PERIOD, freq


def _repeats(got, want):
    whole = got.shape[0] // PERIOD * PERIOD
    return bool((got[:whole].view(-1, *want.shape) == want).all()) and torch.equal(got[whole:], want[:got.shape[0] - whole])


@gpu
def test_rotated():
    n, dim = (1 << 26) - 4, 64
    q, k, _, pos, freq = _inputs(n, dim)
    got = TA.rotate_heads(q, k, pos, freq)
    want = TA.rotate_heads(q[:PERIOD], k[:PERIOD], pos[:PERIOD], freq)
    assert all(_repeats(a, b) for a, b in zip(got, want))
    q, k, _, pos, freq = _inputs(n + 1, dim)
    with pytest.raises(MoldqError, match="2\\^26"):
        TA.rotate_heads(q, k, pos, freq)


@gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_into_the_cache(dim):
    n = ((1 << 35) // dim - 1) // (1 + 512 // dim) // 32 * 32
    q, k, v, pos, freq = _inputs(n, dim)
    page = 4096
    cache = TA.KvCache(-(-n // page), 1, dim, page_tokens=page, dtype=GgmlDType.Q4_0)
    small = TA.KvCache(1, 1, dim, page_tokens=page, dtype=GgmlDType.Q4_0)
    slots = torch.arange(n, device="cuda")
    got, _ = cache.append_rotated(q, k, v, slots, pos, freq)
    want, _ = small.append_rotated(q[:PERIOD], k[:PERIOD], v[:PERIOD], slots[:PERIOD], pos[:PERIOD], freq)
    assert _repeats(got, want)
    whole = n // page
    assert bool((cache.data[:whole * small.data.numel()].view(whole, -1) == small.data).all())
    for a, b in zip(cache.read(slots[whole * page:]), small.read(slots[:n - whole * page])):
        assert torch.equal(a, b)
    q, k, v, pos, freq = _inputs(n + 32, dim)
    with pytest.raises(MoldqError, match="2\\^35"):
        cache.append_rotated(q, k, v, torch.full((n + 32,), -1, device="cuda"), pos, freq)


def test_the_library_refuses_them():
    """On the CPU: before anything is launched, with the limit named."""
    lib, a = _lib.load(), 4096
    rotate = (a, 128, 128, 1, a, 128, 128, 1, 30, 128, (1 << 26) - 3, a, a, None, None, 1e-6, a, a, None)
    assert lib.mq_rotate_heads(*rotate) == _lib.MQ_E_INVALID and b"2^26" in lib.mq_last_error()
    for dim, kv in ((64, 1), (128, 1), (128, 8), (64, 4096)):
        cache = _lib.KvCacheC(a, 4, 8, kv, dim, 64)
        tokens = ((1 << 35) // dim - 1) // (kv + 512 // dim) // 32 * 32 + 1
        into = (a, a, dim, dim, 1, a, dim, dim, a, dim, dim, 30, tokens, a, a, None, None, 1e-6, a, None, None)
        assert lib.mq_kv_cache_append_rotated(ctypes.byref(cache), *into) == _lib.MQ_E_INVALID and b"2^35" in lib.mq_last_error(), (dim, kv)
