"""The paged key/value cache: what append stores and read returns, in every type.

Blocks are compared bit for bit: BF16 with the rounding to nearest even, Q8_0 and Q4_0 with the
framework's reference quantizer (oracle) of the same rows, whose values read returns as
float32.  A bf16 read is those values rounded once more."""
import ctypes

import pytest

torch = pytest.importorskip("torch")
import numpy as np

from mold_amd import GgmlDType, MoldqError, _lib
from mold_amd import text_attention as TA
from oracle import oracle as O

gpu = pytest.mark.gpu
BF = torch.bfloat16
TYPES = [GgmlDType.BF16, GgmlDType.Q8_0, GgmlDType.Q4_0]


def _stored(t, x):
    """float32 values of x's blocks (last axis) by the reference quantizer."""
    if t == GgmlDType.BF16:
        return x.to(BF).float().cpu()
    rows = x.float().cpu().reshape(-1, x.shape[-1]).numpy()
    return torch.from_numpy(np.asarray(O.dequantize(int(t), O.quantize(int(t), rows), *rows.shape))).reshape(x.shape)


def _rows(n, heads, dim, seed=0, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed + 31 * n + dim)
    x = torch.randn((2, n, heads, dim), device="cuda", generator=g) * torch.exp(torch.randn((2, n, heads, 1), device="cuda", generator=g) * 3)
    return x.to(dtype)


@gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("t", TYPES, ids=lambda t: t.name)
@pytest.mark.parametrize("dtype", [torch.float32, BF], ids=["f32", "bf16"])
def test_roundtrip(t, dim, dtype):
    """Any number of tokens at any slots, in any order; the other slots keep what they held."""
    for n, heads, page, pages in [(1, 1, 32, 1), (2, 3, 32, 3), (31, 2, 64, 2), (33, 8, 32, 3), (64, 1, 64, 1), (100, 5, 96, 4), (257, 2, 128, 5)]:
        cache = TA.KvCache(pages, heads, dim, page_tokens=page, dtype=t)
        every = torch.arange(pages * page, device="cuda")
        old = _rows(pages * page, heads, dim, seed=1, dtype=dtype)
        cache.append(old[0], old[1], every)
        slots = torch.randperm(pages * page, device="cuda", generator=torch.Generator(device="cuda").manual_seed(n))[:n]
        new = _rows(n, heads, dim, seed=2, dtype=dtype)
        cache.append(new[0], new[1], slots)
        for i, got in enumerate(cache.read(every, torch.float32)):
            want = _stored(t, old[i])
            want[slots.cpu()] = _stored(t, new[i])
            assert torch.equal(got.cpu(), want), (n, heads, page, "kv"[i])
        for i, got in enumerate(cache.read(slots)):
            assert got.dtype == BF and torch.equal(got.cpu(), _stored(t, new[i]).to(BF)), (n, "kv"[i])


@gpu
@pytest.mark.parametrize("t", TYPES[1:], ids=lambda t: t.name)
def test_block_edges(t):
    """Zero blocks, ties of magnitude with either sign first, halves that round away from zero, one
    large value, and magnitudes whose scale is subnormal or past float16."""
    x = torch.zeros((16, 1, 64))
    x[1, 0, 3], x[1, 0, 40] = 5.0, -5.0
    x[2, 0, 7], x[2, 0, 21] = -3.0, 3.0
    x[3, 0, 21], x[3, 0, 7] = -3.0, 3.0
    x[4, 0, :32] = torch.arange(32) * 0.5 - 7.75
    x[5, 0, :32] = torch.linspace(-127, 127, 32).round() + 0.5
    x[5, 0, 0] = 127.0
    x[6, 0, 31] = 1000.0
    x[7] = 1e-6
    x[8] = 1e-9
    x[9, 0, 5] = 3e6
    x[10, 0, :] = -1.0
    x[11, 0, 15], x[11, 0, 16], x[11, 0, 17] = -2.0, 2.0, -2.0
    x[12, 0, 8], x[12, 0, 9] = 4.0, -4.0
    x[13, 0, 24], x[13, 0, 8] = -4.0, 4.0
    x[14] = torch.randn(64, generator=torch.Generator().manual_seed(1))
    x[15] = -x[14]
    cache = TA.KvCache(1, 1, 64, page_tokens=32, dtype=t)
    slots = torch.arange(16, device="cuda") + 9
    cache.append(x.cuda(), -x.cuda(), slots)
    k, v = cache.read(slots, torch.float32)
    # the same values; a scale past float16 is infinite, and a zero of its block reads as NaN on both sides
    for got, want in ((k, _stored(t, x)), (v, _stored(t, -x))):
        assert torch.isfinite(want).all() == (t == GgmlDType.Q8_0)
        torch.testing.assert_close(got.cpu(), want, rtol=0, atol=0, equal_nan=True)


@gpu
@pytest.mark.parametrize("t", TYPES, ids=lambda t: t.name)
def test_non_finite_values_stay_in_their_block(t):
    for bad in (float("nan"), float("inf"), float("-inf")):
        x = _rows(40, 2, 128, seed=4)
        x[:, 17, 1, 70] = bad
        cache = TA.KvCache(2, 2, 128, page_tokens=32, dtype=t)
        slots = torch.arange(40, device="cuda")
        cache.append(x[0], x[1], slots)
        for i, got in enumerate(cache.read(slots, torch.float32)):
            ok = torch.isfinite(got).cpu()
            where = torch.zeros_like(ok)
            where[17, 1, 70 if t == GgmlDType.BF16 else slice(64, 96)] = True
            assert torch.equal(ok, ~where)
            x[i, 17, 1, 64:96] = 0
            want = _stored(t, x[i])
            want[17, 1, 64:96] = got[17, 1, 64:96].cpu()
            assert torch.equal(got.cpu()[ok], want[ok])


@gpu
@pytest.mark.parametrize("t", TYPES, ids=lambda t: t.name)
def test_slots_outside_the_cache(t):
    cache = TA.KvCache(2, 2, 64, page_tokens=32, dtype=t)
    every = torch.arange(64, device="cuda")
    old, new = _rows(64, 2, 64, seed=1), _rows(5, 2, 64, seed=2)
    cache.append(old[0], old[1], every)
    guard = cache.data.clone()
    outside = torch.tensor([-1, 64, 1 << 40, -(1 << 40), 65], device="cuda")
    cache.append(new[0], new[1], outside)
    assert torch.equal(cache.data, guard)
    k, v = cache.read(outside)
    assert not k.any() and not v.any()
    slots = torch.tensor([3, -1, 63], device="cuda")
    cache.append(new[0, :3], new[1, :3], slots)
    k, _ = cache.read(every, torch.float32)
    want = _stored(t, old[0])
    want[3], want[63] = _stored(t, new[0])[0], _stored(t, new[0])[2]
    assert torch.equal(k.cpu(), want)


@gpu
@pytest.mark.parametrize("t", TYPES, ids=lambda t: t.name)
@pytest.mark.parametrize("first", [64, 1 << 31, 1 << 32, (1 << 63) - 32, -32, -(1 << 63)])
def test_whole_tiles_outside_the_cache(t, first):
    """Slots in the order of a tile, just past the cache's end and as far out as slots go."""
    cache = TA.KvCache(2, 2, 64, page_tokens=32, dtype=t)
    cache.data.fill_(7)
    guard = cache.data.clone()
    slots = torch.arange(32, device="cuda") + first
    new = _rows(32, 2, 64, seed=2)
    cache.append(new[0], new[1], slots)
    assert torch.equal(cache.data, guard)
    k, v = cache.read(slots)
    assert not k.any() and not v.any()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, BF], ids=["f32", "bf16"])
def test_views(dtype):
    """Views of a stacked projection, head-major rows, one head for all, rows off 16 bytes."""
    n = 50
    x = _rows(n, 6, 64, dtype=dtype)[0]
    slots = torch.arange(n, device="cuda")

    def stored(k, v):
        c = TA.KvCache(2, 2, 64, page_tokens=32, dtype=GgmlDType.Q8_0)
        c.append(k, v, slots)
        return torch.cat(c.read(slots, torch.float32))
    k, v = x[:, 2:4], x[:, 4:]
    want = stored(k.contiguous(), v.contiguous())
    assert torch.equal(stored(k, v), want)
    assert torch.equal(stored(*[t.transpose(0, 1).contiguous().transpose(0, 1) for t in (k, v)]), want)
    assert torch.equal(stored(*[torch.nn.functional.pad(t, (1, 4))[:, :, 1:65] for t in (k, v)]), want)
    assert torch.equal(stored(*[t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v)]), want)
    one = x[:, 2:3].expand(-1, 2, -1)
    assert torch.equal(stored(one, v), stored(one.contiguous(), v))
    c = TA.KvCache(2, 2, 64, page_tokens=32, dtype=GgmlDType.Q8_0)
    c.append(k, v, torch.stack([slots, slots], 1)[:, 0])       # strided slots
    assert torch.equal(torch.cat(c.read(slots, torch.float32)), want)


@gpu
def test_pages_past_32_bits():
    """A cache of more than 4 GB: its last page is where it should be and no other."""
    pages = 36000
    cache = TA.KvCache(pages, 4, 128, page_tokens=64, dtype=GgmlDType.BF16)
    assert cache.data.numel() > 1 << 32
    new = _rows(64, 4, 128, seed=3, dtype=BF)
    far = torch.arange(64, device="cuda") + (pages - 1) * 64
    near = torch.arange(64, device="cuda")
    cache.append(new[0], new[1], far)
    cache.append(new[1], new[0], near)
    assert all(torch.equal(a, b) for a, b in zip(cache.read(far), (new[0], new[1])))
    assert all(torch.equal(a, b) for a, b in zip(cache.read(near), (new[1], new[0])))


@gpu
def test_rows_past_32_bits():
    """Rows 2^22 elements apart, 1100 of them: 9 GB in bf16; and 2^24 apart, which are copied."""
    new = _rows(1100, 2, 64, seed=6, dtype=BF)
    slots = torch.arange(1100, device="cuda")
    want = TA.KvCache(35, 2, 64, page_tokens=32)
    want.append(new[0], new[1], slots)
    for n, step in ((1100, 1 << 22), (40, 1 << 24)):
        far = torch.empty((n - 1) * step + 256, dtype=BF, device="cuda").as_strided((n, 4, 64), (step, 64, 1))
        far.copy_(torch.cat([new[0], new[1]], 1)[:n])
        cache = TA.KvCache(35, 2, 64, page_tokens=32)
        cache.append(far[:, :2], far[:, 2:], slots[:n])
        assert all(torch.equal(a, b[:n]) for a, b in zip(cache.read(slots[:n]), want.read(slots)))
        del far


@gpu
def test_slots_of_positions_and_streams():
    cache = TA.KvCache(6, 2, 64, page_tokens=32)
    table = torch.tensor([[4, 1], [0, 5]], dtype=torch.int32, device="cuda")
    pos = torch.tensor([[0, 31, 32, 63], [-1, 5, 40, -7]], device="cuda")
    assert cache.slots(table, pos).tolist() == [[128, 159, 32, 63], [-1, 5, 168, -1]]
    x = _rows(4, 2, 64, dtype=BF)
    slots = cache.slots(table, pos)[0]
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()) as _:
        cache.append(x[0], x[1], slots)
        k, v = cache.read(slots, torch.float32)
        torch.cuda.current_stream().synchronize()
    assert torch.equal(k.cpu(), _stored(GgmlDType.Q8_0, x[0])) and torch.equal(v.cpu(), _stored(GgmlDType.Q8_0, x[1]))


@gpu
def test_refused_calls():
    cache = TA.KvCache(2, 2, 64, page_tokens=32)
    k, slots = torch.zeros((3, 2, 64), device="cuda"), torch.arange(3, device="cuda")
    for args in [(k, k.to(BF), slots), (k.half(), k.half(), slots), (k[:2], k, slots), (k, k, slots.int()), (k, k, slots.cpu()), (k.cpu(), k, slots),
                 (k[:, :1], k, slots), (k[..., :32], k, slots), (k, k, slots[None]), (k.requires_grad_(True), k, slots)]:
        with pytest.raises(ValueError):
            cache.append(*args)
    for args in [(slots.int(),), (slots.cpu(),), (slots, torch.float16)]:
        with pytest.raises(ValueError):
            cache.read(*args)
    k = k.detach()
    cache.append(k[:0], k[:0], slots[:0])
    assert cache.read(slots[:0])[0].shape == (0, 2, 64)
    for kw in (dict(head_dim=96), dict(page_tokens=48), dict(page_tokens=0), dict(dtype=GgmlDType.Q4_K), dict(kv_heads=0), dict(pages=-1)):
        with pytest.raises(ValueError):
            TA.KvCache(**{"pages": 2, "kv_heads": 2, **kw})


def _cache(dtype=8, kv=2, dim=64, page=32, pages=3, data=4096):
    return _lib.KvCacheC(data, pages, dtype, kv, dim, page)


def test_sizes():
    lib = _lib.load()
    for t, per in ((30, 128.0), (8, 68.0), (2, 36.0)):
        for dim in (64, 128):
            c = _cache(t, 3, dim, 96, 5)
            assert lib.mq_kv_cache_size(ctypes.byref(c)) == int(5 * 3 * 3 * per * dim)
    for bad in (dict(dtype=12), dict(kv=0), dict(kv=5000), dict(dim=32), dict(page=33), dict(page=0), dict(page=65568), dict(pages=-1)):
        assert lib.mq_kv_cache_size(ctypes.byref(_cache(**bad))) == 0
    assert lib.mq_kv_cache_size(None) == 0
    big = _cache(30, 8, 128, 65536, 1 << 20)
    assert lib.mq_kv_cache_size(ctypes.byref(big)) == (1 << 20) * 8 * 2048 * 16384


def test_argument_checks():
    lib = _lib.load()

    def append(c=None, k=4096, ks=(128, 64), v=4096, vs=(128, 64), dt=30, n=3, slots=4096):
        c = c or _cache()
        return lib.mq_kv_cache_append(ctypes.byref(c), k, *ks, v, *vs, dt, n, slots, None)

    def read(c=None, slots=4096, n=3, k=4096, v=4096, dt=30):
        c = c or _cache()
        return lib.mq_kv_cache_read(ctypes.byref(c), slots, n, k, v, dt, None)
    for kw in (dict(k=None), dict(slots=None), dict(k=4100), dict(slots=4100), dict(ks=(-128, 64)), dict(vs=(128, 60)), dict(vs=(1 << 24, 64)), dict(dt=1), dict(n=-1),
               dict(n=1 << 31), dict(c=_cache(page=16)), dict(c=_cache(data=4100)), dict(c=_cache(data=None)), dict(ks=(2, 64), dt=0)):
        assert append(**kw) == -1, kw
    for kw in (dict(k=None), dict(v=4098), dict(slots=None), dict(dt=8), dict(n=-5), dict(c=_cache(dtype=3)), dict(c=_cache(data=4098))):
        assert read(**kw) == -1, kw
    with pytest.raises(MoldqError):
        _lib.check(append(k=None))
    assert lib.mq_kv_cache_append(None, None, 0, 0, None, 0, 0, 0, 0, None, None) == -1
    assert append(n=0, k=None) == 0 and read(n=0, k=None) == 0
