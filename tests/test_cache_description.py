"""A cache's description whose size passes 64 bits is no description: its size is 0 and every
entry point refuses it.  A size modulo 2^64 would be a buffer that its slots lie outside of."""
import ctypes

import pytest

from mold_amd import GgmlDType, _lib

# type, heads, head_dim, page_tokens, pages
WRAPPING = [(2, 4095, 64, 65504, 955136626),               # 266207744 modulo 2^64
            (30, 4096, 128, 65536, (1 << 31) - 1),         # 2^68 bytes and less
            (30, 4096, 128, 65536, 1 << 27),               # 2^64
            (30, 4096, 128, 65536, 1 << 26),               # 2^63: a pointer difference no longer
            (8, 4096, 128, 65536, 1 << 30)]


def _cache(t, heads, dim, page, pages):
    return _lib.KvCacheC(4096, pages, t, heads, dim, page)


@pytest.mark.parametrize("what", WRAPPING)
def test_wrapping_sizes_are_refused(what):
    lib, c = _lib.load(), _cache(*what)
    ref, h, d = ctypes.byref(c), what[1], what[2]
    assert lib.mq_kv_cache_size(ref) == 0
    assert lib.mq_kv_cache_append(ref, 4096, h * d, d, 4096, h * d, d, 30, 1, 4096, None) == _lib.MQ_E_INVALID
    assert lib.mq_kv_cache_read(ref, 4096, 1, 4096, 4096, 30, None) == _lib.MQ_E_INVALID
    assert lib.mq_cache_attention(ref, 4096, h * d, d, 1, h, 4096, 1, 1, 4096, 0.125, 1 << 24, h * d, d, None, 0, None) == _lib.MQ_E_INVALID
    assert lib.mq_cache_attention_scratch_size(ref, 64, h, 1 << 10) == 0


def test_the_largest_sizes_are_whole():
    lib = _lib.load()
    for t, per in ((30, 128), (8, 68), (2, 36)):
        pages = ((1 << 63) - 1) // (4096 * 2048 * per * 128)
        c = _cache(t, 4096, 128, 65536, pages)
        assert lib.mq_kv_cache_size(ctypes.byref(c)) == pages * 4096 * 2048 * per * 128
        c.pages = pages + 1
        assert lib.mq_kv_cache_size(ctypes.byref(c)) == 0


def test_the_python_cache_refuses_them():
    TA = pytest.importorskip("mold_amd.text_attention")
    for t, heads, dim, page, pages in WRAPPING:
        with pytest.raises(ValueError):
            TA.KvCache(pages, heads, dim, page, GgmlDType(t))
