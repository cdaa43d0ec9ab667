"""Head norms and rotation of q and k (rotate_heads), and the same on the way into the paged cache
(KvCache.append_rotated), against the formulas in float64.

Bounds: a result is rounded once to bf16, at most 2^-8 of its value off.  Before that, in float32: the
sum of D <= 128 squares, each product and sum off by 2^-24 of it, D 2^-24 = 2^-17 in all at most,
half of that in the root; the root, two products, the rotation's two products and its sum, each at most 2^-23: 2^-20
together; sine and cosine of an angle that is off by 2^-24 turns at the farthest positions (2^28.4
turns in 64 bits, whose product is rounded twice: 6.3 * 2^-24), rounded to f32 themselves, below 2^-20
together.  2^-16 (|y_i| + |y_(i + D/2)|) holds them all."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from mold_amd import GgmlDType, MoldqError, _lib
from mold_amd import text_attention as TA

gpu = pytest.mark.gpu
BF = torch.bfloat16
TYPES = [GgmlDType.BF16, GgmlDType.Q8_0, GgmlDType.Q4_0]


def _inputs(n, heads, kv, dim, dtype, seed=0, far=4000):
    """One projection's output, its parts side by side; positions; frequencies; two norms."""
    g = torch.Generator(device="cuda").manual_seed(seed + 7 * n + dim)
    qkv = (torch.randn((n, heads + 2 * kv, dim), device="cuda", generator=g) * torch.exp(torch.randn((n, heads + 2 * kv, 1), device="cuda", generator=g))).to(dtype)
    pos = torch.randint(0, far, (n,), device="cuda", generator=g)
    freq = 1e6 ** (-torch.arange(dim // 2, device="cuda", dtype=torch.float32) / (dim // 2))
    qw, kw = 1 + 0.2 * torch.randn((2, dim), device="cuda", generator=g)
    return qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:], pos, freq, qw, kw


def _exact(x, pos, freq, weight, eps):
    """float64 result, and |y_i| + |y_(i + D/2)| for each value."""
    x = x.double()
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    a, b = x.chunk(2, -1)
    angle = (pos.double()[:, None] * freq.double())[:, None]
    size = a.abs() + b.abs()
    return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], -1), torch.cat([size, size], -1)


def _check(got, x, pos, freq, weight, eps=1e-6):
    assert got.dtype == BF and got.shape == x.shape
    want, size = _exact(x, pos, freq, weight, eps)
    off = (got.double() - want).abs() - 2.0 ** -8 * want.abs() - 2.0 ** -16 * size
    assert off.numel() == 0 or off.max() <= 0, off.max()


@gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("norm", ["none", "q", "both"])
def test_heads(dim, dtype, norm):
    """Heads that fill a wave's pass, leave a part of one, or are one; a token to a few thousand."""
    for n, heads, kv in [(1, 1, 1), (1, 32, 8), (3, 7, 7), (33, 16, 2), (500, 5, 1), (2049, 9, 3), (4000, 28, 4)]:
        q, k, _, pos, freq, qw, kw = _inputs(n, heads, kv, dim, dtype)
        qw, kw = (None, None) if norm == "none" else (qw, None) if norm == "q" else (qw, kw)
        gq, gk = TA.rotate_heads(q, k, pos, freq, qw, kw, eps=1e-5)
        _check(gq, q, pos, freq, qw, 1e-5)
        _check(gk, k, pos, freq, kw, 1e-5)


@gpu
def test_positions_as_far_as_they_go():
    """Angles keep their fraction of a turn: 2^31 positions are 2^29 turns at the first frequency."""
    n = 64
    q, k, _, _, freq, qw, kw = _inputs(n, 4, 2, 128, torch.float32)
    for pos in (torch.zeros(n, dtype=torch.int64), torch.arange(n) + (1 << 31) - n, (1 << 24) + torch.arange(n) * 65537, -torch.arange(n)):
        pos = pos.cuda()
        gq, gk = TA.rotate_heads(q, k, pos, freq, qw, kw)
        _check(gq, q, pos, freq, qw)
        _check(gk, k, pos, freq, kw)
    gq, _ = TA.rotate_heads(q, k, torch.zeros(n, dtype=torch.int64, device="cuda"), freq)
    assert torch.equal(gq, q.to(BF))


@gpu
def test_values_at_the_ends():
    """Zero heads, tiny and large ones; what is not a number stays in its head."""
    q, k, _, pos, freq, qw, kw = _inputs(40, 4, 2, 128, torch.float32)
    q, k = q.clone(), k.clone()
    q[3], q[5, 1], q[6, 2], k[7, 0] = 0, q[5, 1] * 1e-12, q[6, 2] * 1e15, 0
    _check(TA.rotate_heads(q, k, pos, freq, qw, kw)[0], q, pos, freq, qw)
    want = TA.rotate_heads(q, k, pos, freq, qw, kw)
    for bad in (float("nan"), float("inf")):
        q2, k2 = q.clone(), k.clone()
        q2[9, 1, 70], k2[11, 1, 3] = bad, bad
        got = TA.rotate_heads(q2, k2, pos, freq, qw, kw)
        for g, w, at in zip(got, want, ((9, 1), (11, 1))):
            same = torch.ones(g.shape[:2], dtype=torch.bool, device="cuda")
            same[at] = False
            assert torch.equal(g[same], w[same]) and torch.isnan(g[at]).any()
        got = TA.rotate_heads(q2, k2, pos, freq)         # without a norm it stays in its pair
        bad_at = torch.nonzero(~torch.isfinite(got[0])).tolist()
        assert bad_at and all(at in ([9, 1, 70], [9, 1, 6]) for at in bad_at)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, BF], ids=["f32", "bf16"])
def test_strides_and_alignment(dtype):
    """Views of any strides, starting anywhere, give what their packed copies give."""
    n, heads, kv, dim = 37, 6, 3, 64
    q, k, _, pos, freq, qw, kw = _inputs(n, heads, kv, dim, dtype)
    want = TA.rotate_heads(q.contiguous(), k.contiguous(), pos, freq, qw, kw)
    wide = torch.zeros((n, heads + 1, dim + 24), dtype=dtype, device="cuda")
    wide[:, 1:, 16:16 + dim] = q
    shifted = torch.empty(q.numel() + 8, dtype=dtype, device="cuda")[1:1 + q.numel()].view(q.shape).copy_(q)
    by_head = q.transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.zeros((n, heads, dim + 1), dtype=dtype, device="cuda")
    odd[..., 1:] = q
    for view in (wide[:, 1:, 16:16 + dim], shifted, by_head, odd[..., 1:], q.expand(n, heads, dim)):
        got = TA.rotate_heads(view, k, pos, freq, qw, kw)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    every = torch.zeros((n, 2), dtype=torch.int64, device="cuda")
    every[:, 1] = pos
    pairs = torch.stack([freq, freq], 1)
    got = TA.rotate_heads(q, k, every[:, 1], pairs[:, 1], torch.stack([qw, qw], 1)[:, 0], kw)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    one = q[:1].expand(n, heads, dim)                         # a token stride of 0
    got = TA.rotate_heads(one, k, pos, freq, qw, kw)[0]
    _check(got, one, pos, freq, qw)


@gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("t", TYPES, ids=lambda t: t.name)
@pytest.mark.parametrize("dtype", [torch.float32, BF], ids=["f32", "bf16"])
def test_into_the_cache(t, dim, dtype):
    """The cache's bytes and both results are those of the separate calls; other slots keep what they held."""
    for n, heads, kv, page in [(1, 4, 1, 32), (31, 8, 8, 32), (32, 3, 2, 64), (48, 16, 8, 64), (130, 7, 1, 96), (2000, 12, 4, 128)]:
        q, k, v, pos, freq, qw, kw = _inputs(n, heads, kv, dim, dtype)
        pages = -(-n // page) + 2
        for kind in ("runs", "scattered", "outside"):
            slots = torch.arange(n, device="cuda") + page if kind == "runs" else torch.randperm(pages * page, device="cuda")[:n]
            if kind == "outside":
                slots[::3] = torch.tensor([-1, pages * page, 1 << 40], device="cuda").repeat(n)[:slots[::3].shape[0]]
            one, two = (TA.KvCache(pages, kv, dim, page_tokens=page, dtype=t) for _ in range(2))
            one.data.fill_(37)
            two.data.fill_(37)
            want = TA.rotate_heads(q, k, pos, freq, qw, kw)
            if dtype == BF:
                one.append(want[1], v, slots)
            else:                                             # bf16 keys beside f32 values: f32 holds both
                one.append(want[1].float(), v, slots)
            got = two.append_rotated(q, k, v, slots, pos, freq, qw, kw, keys=True)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), (n, kind)
            assert torch.equal(one.data, two.data), (n, kind)
            three = TA.KvCache(pages, kv, dim, page_tokens=page, dtype=t)
            three.data.fill_(37)
            got = three.append_rotated(q, k, v, slots, pos, freq, qw, kw)
            assert got[1] is None and torch.equal(got[0], want[0]) and torch.equal(three.data, two.data)


@gpu
def test_no_tokens_and_no_pages():
    q, k, v, pos, freq, qw, kw = _inputs(5, 4, 2, 64, BF)
    got = TA.rotate_heads(q[:0], k[:0], pos[:0], freq)
    assert got[0].shape == (0, 4, 64) and got[1].shape == (0, 2, 64)
    slots = torch.arange(5, device="cuda")
    cache = TA.KvCache(0, 2, 64, page_tokens=32)
    got = cache.append_rotated(q, k, v, slots, pos, freq, keys=True)
    want = TA.rotate_heads(q, k, pos, freq)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert cache.append_rotated(q[:0], k[:0], v[:0], slots[:0], pos[:0], freq)[0].shape == (0, 4, 64)


@gpu
def test_captured_and_on_other_streams():
    """A graph reads what its buffers hold at each replay."""
    q, k, v, pos, freq, qw, kw = _inputs(70, 8, 2, 128, BF)
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    slots = torch.arange(70, device="cuda") + 9
    cache, plain = (TA.KvCache(4, 2, 128, page_tokens=32) for _ in range(2))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        cache.append_rotated(q, k, v, slots, pos, freq, qw, kw)
        with torch.cuda.graph(graph, stream=s):
            out, keys = cache.append_rotated(q, k, v, slots, pos, freq, qw, kw, keys=True)
            alone = TA.rotate_heads(q, k, pos, freq, qw, kw)
    torch.cuda.current_stream().wait_stream(s)
    cache.data.zero_()                                        # the first call has written to it
    plain.data.zero_()
    for i in range(4):
        x = _inputs(70, 8, 2, 128, BF, seed=i + 1)
        q.copy_(x[0]), k.copy_(x[1]), v.copy_(x[2]), pos.copy_(x[3])
        slots.copy_(torch.randperm(128, device="cuda")[:70])
        want = plain.append_rotated(q, k, v, slots, pos, freq, qw, kw, keys=True)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((out, keys, *alone), want * 2):
            assert torch.equal(a, b), i
        assert torch.equal(cache.data, plain.data), i


@gpu
def test_refusals():
    q, k, v, pos, freq, qw, kw = _inputs(8, 4, 2, 64, BF)
    slots, cache = torch.arange(8, device="cuda"), TA.KvCache(1, 2, 64, page_tokens=32)
    ok = dict(q=q, k=k, positions=pos, inv_freq=freq, q_weight=qw, k_weight=kw)
    for change in (dict(q=q.half()), dict(q=q.float()), dict(q=q[:7]), dict(q=q[:, :0]), dict(q=q[..., :32]), dict(q=q[0]), dict(q=q.cpu()), dict(k=k[..., :32]),
                   dict(k=k[:, :0]), dict(positions=pos.int()), dict(positions=pos[:7]), dict(positions=pos.cpu()), dict(inv_freq=freq[:16]),
                   dict(inv_freq=freq.double()), dict(q_weight=qw.to(BF)), dict(k_weight=kw[:32]), dict(q_weight=qw.cpu()),
                   dict(q=q.clone().requires_grad_()), dict(k_weight=kw.clone().requires_grad_()), dict(inv_freq=freq.clone().requires_grad_())):
        with pytest.raises(ValueError):
            TA.rotate_heads(**{**ok, **change})
        with pytest.raises(ValueError):
            cache.append_rotated(**{**ok, **change}, v=v, slots=slots)
    for change in (dict(v=v.float()), dict(v=v[:, :1]), dict(k=k[:, :1]), dict(slots=slots.int()), dict(slots=slots[:7]), dict(slots=slots.cpu())):
        with pytest.raises(ValueError):
            cache.append_rotated(**{**ok, "v": v, "slots": slots, **change})
    for eps in (-1e-6, float("nan"), float("inf")):
        with pytest.raises(MoldqError):
            TA.rotate_heads(**ok, eps=eps)
    with torch.no_grad():
        TA.rotate_heads(**{**ok, "q": q.clone().requires_grad_()})


def test_refusals_of_the_library():
    """On the CPU: every fault is found before anything is launched."""
    lib = _lib.load()
    a, bad = 4096, _lib.MQ_E_INVALID
    rotate = dict(q=a, qt=512, qh=128, heads=4, k=a, kt=256, kh=128, kv=2, x=30, dim=128, n=3, pos=a, freq=a, qw=a, kw=a, eps=1e-6, qo=a, ko=a, stream=None)
    changes = [dict(q=None), dict(k=None), dict(pos=None), dict(freq=None), dict(qo=None), dict(ko=None), dict(q=a + 8), dict(k=a + 2), dict(qo=a + 4),
               dict(ko=a + 8), dict(freq=a + 4), dict(qw=a + 4), dict(kw=a + 8), dict(pos=a + 4), dict(qt=4), dict(qh=-8), dict(kt=1 << 24), dict(kh=3), dict(heads=0),
               dict(kv=0), dict(heads=65537), dict(x=1), dict(dim=96), dict(n=-1), dict(n=1 << 31), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")),
               dict(n=(1 << 31) - 1, heads=65536)]
    for change in changes:
        assert lib.mq_rotate_heads(*{**rotate, **change}.values()) == bad, change
    assert lib.mq_rotate_heads(*{**rotate, "n": 0, "q": None}.values()) == 0
    cache = _lib.KvCacheC(a, 4, 8, 2, 128, 64)
    into = dict(slots=a, q=a, qt=512, qh=128, heads=4, k=a, kt=256, kh=128, v=a, vt=256, vh=128, x=30, n=3, pos=a, freq=a, qw=a, kw=a, eps=1e-6, qo=a,
                ko=None, stream=None)
    for change in [c for c in changes if set(c) <= set(into) and c != dict(ko=None)] + [dict(slots=None), dict(slots=a + 4), dict(v=None), dict(v=a + 8), dict(vt=4), dict(vh=1 << 24)]:
        assert lib.mq_kv_cache_append_rotated(ctypes.byref(cache), *{**into, **change}.values()) == bad, change
    for field, value in (("data", None), ("data", a + 8), ("pages", -1), ("dtype", 12), ("head_dim", 96), ("kv_heads", 0), ("page_tokens", 33)):
        c = _lib.KvCacheC(a, 4, 8, 2, 128, 64)
        setattr(c, field, value)
        assert lib.mq_kv_cache_append_rotated(ctypes.byref(c), *into.values()) == bad, field
    assert lib.mq_kv_cache_append_rotated(None, *into.values()) == bad
