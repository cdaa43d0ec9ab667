"""mq_cache_attention (attention of one new token per sequence over the paged cache) against
float64 attention over the values the cache holds: tile and page edges, runs that split or span
sequences, groups of heads, garbage beside what a sequence owns, and its refusals.

The bound on the relative error is that of the roundings to bf16 of the probabilities (with a
value block's scale) and of the output, 1.66e-3 each on average, 2.4e-3 together (keys and
values enter exactly); 3e-3 is asserted over a whole output."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from mold_amd import GgmlDType, MoldqError, _lib
from mold_amd import text_attention as TA
from tests.test_build_checks import HIPCC, _asm, _functions

gpu = pytest.mark.gpu
BOUND = 3e-3
BF = torch.bfloat16
TYPES = [GgmlDType.BF16, GgmlDType.Q8_0, GgmlDType.Q4_0]
I32_JUNK = [-1, 1 << 30, -(1 << 31)]


class _Batch:
    """A cache filled with NaN bytes, sequences of `lengths` in pages in no order, and a table
    whose entries past a sequence's pages name no page."""

    def __init__(self, lengths, heads, kv, dim, t, page=64, seed=0, extra=2, sharp=1.0):
        g = torch.Generator(device="cuda").manual_seed(seed + 13 * sum(lengths) + dim + heads)
        per = [-(-n // page) for n in lengths]
        self.lengths, self.page = lengths, page
        self.cache = TA.KvCache(max(1, sum(per) + extra), kv, dim, page_tokens=page, dtype=t)
        self.cache.data.fill_(255)
        order = torch.randperm(self.cache.pages, generator=torch.Generator().manual_seed(seed)).tolist()
        width = max(per, default=0) + 1
        rows, self.slots = [], []
        for n, p in zip(lengths, per):
            mine, order = order[:p], order[p:]
            rows.append(mine + [I32_JUNK[i % 3] for i in range(width - p)])
            at = torch.arange(n)
            self.slots.append((torch.tensor(mine + [0], dtype=torch.int64)[at // page] * page + at % page).cuda())
        self.table = torch.tensor(rows, dtype=torch.int64).to(torch.int32).reshape(len(lengths), width).cuda()
        self.len = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        every = torch.cat(self.slots) if lengths else torch.empty(0, dtype=torch.int64, device="cuda")
        x = torch.randn((2, every.numel(), kv, dim), device="cuda", generator=g)
        self.cache.append(x[0], x[1], every)
        self.q = (torch.randn((len(lengths), heads, dim), device="cuda", generator=g) * sharp).to(BF)

    def run(self, **kw):
        return self.cache.attend(self.q, self.table, self.len, **kw)

    def ref(self, scale=None):
        n, heads, dim = self.q.shape
        group, scale = heads // self.cache.kv_heads, dim ** -0.5 if scale is None else scale
        out = torch.zeros((n, heads, dim), dtype=torch.float64)
        for b, slots in enumerate(self.slots):
            if slots.numel():
                k, v = (t.double().repeat_interleave(group, 1).transpose(0, 1).contiguous()
                        for t in self.cache.read(slots, torch.float32))
                s = (k @ self.q[b].double().unsqueeze(2)).squeeze(2) * scale
                out[b] = (torch.softmax(s, -1).unsqueeze(1) @ v).squeeze(1).cpu()
        return out


def _err(out, ref):
    return ((out.double().cpu() - ref).norm() / ref.norm()).item()


@gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("t", TYPES, ids=lambda t: t.name)
def test_lengths(t, dim):
    for n in (1, 2, 31, 32, 33, 63, 64, 65, 96, 97, 127, 129, 500, 1025):
        b = _Batch([n], 4, 2, dim, t, page=32 if n % 2 else 64)
        out = b.run()
        assert _err(out, b.ref()) < BOUND, n
        assert torch.equal(out, b.run()), n


@gpu
@pytest.mark.parametrize("t", TYPES, ids=lambda t: t.name)
@pytest.mark.parametrize("heads,kv", [(1, 1), (6, 2), (7, 1), (16, 1), (17, 1), (40, 1), (32, 8), (20, 20)])
def test_groups(heads, kv, t):
    """Groups of one, odd ones, one of exactly a matrix instruction's columns, and larger ones."""
    for dim in (64, 128):
        b = _Batch([70, 1, 200], heads, kv, dim, t, page=96)
        assert _err(b.run(), b.ref()) < BOUND, dim


@gpu
@pytest.mark.parametrize("t", TYPES, ids=lambda t: t.name)
def test_ragged_batches(t):
    """Runs that end inside a sequence, span several, and skip empty ones; more than 64 sequences."""
    g = torch.Generator().manual_seed(7)
    for count, top, page, heads, kv in [(5, 300, 32, 8, 2), (64, 400, 64, 8, 4), (65, 200, 32, 4, 1), (200, 130, 32, 8, 8), (130, 900, 96, 16, 8)]:
        lengths = (torch.randint(0, top, (count,), generator=g) * (torch.rand(count, generator=g) > 0.3)).tolist()
        b = _Batch(lengths, heads, kv, 64, t, page=page)
        out, ref = b.run(), b.ref()
        assert _err(out, ref) < BOUND, count
        for i, n in enumerate(lengths):
            assert n or not out[i].any(), i
        assert torch.equal(out, b.run())
    b = _Batch([0] * 70 + [45] + [0] * 80, 4, 2, 64, t)
    assert _err(b.run(), b.ref()) < BOUND


@gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("t", TYPES, ids=lambda t: t.name)
@pytest.mark.parametrize("count,heads,kv,longest", [(63, 16, 8, 300), (64, 16, 8, 300), (127, 8, 8, 1000), (128, 8, 8, 1000), (128, 8, 8, 2016),
                                                    (128, 8, 8, 2017), (9, 120, 60, 1984), (31, 51, 17, 100)])
def test_many_rows(t, dim, count, heads, kv, longest):
    """About 512 and 1024 rows and tables of 32 and 64 tiles, where the split over workgroups changes."""
    g = torch.Generator().manual_seed(count + longest)
    lengths = [longest] + torch.randint(0, min(longest, 400), (count - 1,), generator=g).tolist()
    b = _Batch(lengths, heads, kv, dim, t, page=32)
    out = b.run()
    assert _err(out, b.ref()) < BOUND
    assert torch.equal(out, b.run())
    for i, n in enumerate(lengths):
        assert n or not out[i].any(), i


@gpu
@pytest.mark.parametrize("t", TYPES, ids=lambda t: t.name)
@pytest.mark.parametrize("lengths,heads,kv", [([40000], 4, 1), ([70001, 3, 20000], 8, 2), ([9000] * 6, 8, 8)])
def test_long_contexts(lengths, heads, kv, t):
    """Hundreds of shares a sequence, tables of more than 64 pages."""
    b = _Batch(lengths, heads, kv, 128, t, page=32)
    assert _err(b.run(), b.ref()) < BOUND


@gpu
@pytest.mark.parametrize("sharp,scale", [(0.0, None), (30.0, None), (1.0, 0.7), (1.0, 1e-4)])
@pytest.mark.parametrize("t", TYPES, ids=lambda t: t.name)
def test_flat_and_one_hot_rows(t, sharp, scale):
    b = _Batch([300, 77, 1500], 4, 2, 128, t, sharp=sharp)
    assert _err(b.run(scale=scale), b.ref(scale)) < BOUND


@gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("t", TYPES, ids=lambda t: t.name)
def test_what_lies_past_a_length_is_not_seen(t, bad):
    """Tokens after the length, in its own last tile and page, change no bit of the result."""
    for dim in (64, 128):
        b = _Batch([200, 333], 4, 2, dim, t, page=64)
        whole = b.run()
        assert _err(whole, b.ref()) < BOUND
        full_slots = b.slots
        for cut in ([199, 332], [193, 321], [161, 300], [1, 33]):
            b.len.copy_(torch.tensor(cut, dtype=torch.int32))
            b.slots = [s[:n] for s, n in zip(full_slots, cut)]
            want = b.run()
            assert _err(want, b.ref()) < BOUND, cut
            past = torch.cat([s[n:] for s, n in zip(full_slots, cut)])
            keep = b.cache.data.clone()
            x = torch.full((past.numel(), 2, dim), bad, device="cuda")
            b.cache.append(x, x, past)
            assert torch.equal(b.run(), want), cut
            b.cache.data.copy_(keep)


@gpu
def test_non_finite_values_that_are_seen():
    b = _Batch([100, 100], 4, 2, 64, GgmlDType.BF16)
    clean = b.run()
    k, v = b.cache.read(b.slots[1])
    v[40, 1, 9], v[41, 1, 10] = float("nan"), float("inf")
    b.cache.append(k, v, b.slots[1])
    out = b.run()
    assert torch.equal(out[0], clean[0]) and torch.equal(out[1, :2], clean[1, :2])
    assert torch.isnan(out[1, 2:, 9]).all() and (out[1, 2:, 10] == float("inf")).all()
    rest = [c for c in range(64) if c not in (9, 10)]
    assert torch.equal(out[1, 2:][:, rest], clean[1, 2:][:, rest])
    k[40, 0, 3] = float("nan")
    b.cache.append(k, v, b.slots[1])
    assert torch.isnan(b.run()[1, :2]).all()


@gpu
@pytest.mark.parametrize("t", [GgmlDType.BF16, GgmlDType.Q8_0], ids=lambda t: t.name)
def test_pages_outside_the_cache(t):
    """A sequence that names a page outside the cache, or more tokens than its table, reads as NaN;
    the others keep every bit.  No memory outside the cache is touched."""
    for junk in I32_JUNK + [None]:
        b = _Batch([100, 150, 5000, 40], 4, 2, 64, t, page=32)
        want = b.run()
        b.table[1, 2] = b.cache.pages if junk is None else junk
        b.len[3] = b.table.shape[1] * 32 + 1
        b.table[3] = b.table[2]
        out = b.run()
        assert torch.equal(out[0], want[0]) and torch.equal(out[2], want[2])
        assert torch.isnan(out[1]).all() and torch.isnan(out[3]).all()
    b.len[3], b.len[1] = -5, 0
    out = b.run()
    assert not out[1].any() and not out[3].any() and torch.equal(out[2], want[2])
    none = torch.zeros((4, 0), dtype=torch.int32, device="cuda")
    b.len.copy_(torch.tensor([0, 3, 0, -1], dtype=torch.int32))
    out = b.cache.attend(b.q, none, b.len)
    assert torch.isnan(out[1]).all() and not out[[0, 2, 3]].any()


@gpu
def test_views_and_strided_out():
    b = _Batch([100, 3, 64], 4, 2, 64, GgmlDType.Q8_0)
    want = b.run()
    q = b.q
    stacked = torch.cat([q, torch.zeros_like(q)], 1)
    for view in (stacked[:, :4], q.transpose(0, 1).contiguous().transpose(0, 1), torch.nn.functional.pad(q, (1, 2))[:, :, 1:65]):
        b.q = view
        assert torch.equal(b.run(), want)
    buf = torch.full((3, 6, 80), 3.0, dtype=BF, device="cuda")
    view = buf[:, 1:5, 8:72]
    assert b.run(out=view) is view and torch.equal(view, want)
    view.fill_(3.0)
    assert bool((buf == 3.0).all())
    odd = torch.full((3, 4, 67), 3.0, dtype=BF, device="cuda")
    assert torch.equal(b.run(out=odd[:, :, 1:65]), want) and bool((odd[:, :, 65:] == 3.0).all())
    b.q = stacked[:, :4]
    assert torch.equal(b.run(out=stacked[:, :4]), want)
    b.q = q
    wide = torch.full((3, 20), -1, dtype=torch.int32, device="cuda")
    wide[:, :b.table.shape[1]] = b.table
    b.table = wide[:, :b.table.shape[1]]
    assert torch.equal(b.run(), want)
    b.table = b.table.t().contiguous().t()
    b.len = torch.stack([b.len, b.len], 1)[:, 0]
    assert torch.equal(b.run(), want)


@gpu
def test_cache_past_32_bits():
    page = 64
    cache = TA.KvCache(36000, 4, 128, page_tokens=page, dtype=GgmlDType.BF16)
    cache.data[:1 << 20].fill_(255)
    small = TA.KvCache(3, 4, 128, page_tokens=page, dtype=GgmlDType.BF16)
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v = torch.randn((2, 150, 4, 128), device="cuda", generator=g)
    q = torch.randn((1, 8, 128), device="cuda", generator=g).to(BF)
    n = torch.tensor([150], dtype=torch.int32, device="cuda")
    outs = []
    for c, pages in ((cache, [35999, 17000, 35998]), (small, [0, 1, 2])):
        table = torch.tensor([pages], dtype=torch.int32, device="cuda")
        c.append(k, v, c.slots(table, torch.arange(150, device="cuda")[None])[0])
        outs.append(c.attend(q, table, n))
    assert torch.equal(*outs) and torch.isfinite(outs[0]).all()


@gpu
def test_other_streams_and_graphs():
    """A captured call reads lengths, table and cache anew at each replay."""
    b = _Batch([100, 700, 1, 0], 8, 2, 128, GgmlDType.Q8_0, page=32)
    want = b.run()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = b.run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            kept = b.run()
    s.synchronize()
    assert torch.equal(got, want)
    for i, lengths in enumerate(([100, 700, 1, 0], [99, 650, 0, 0], [1, 1, 1, 0], [0, 0, 0, 0], [64, 512, 1, 0])):
        b.len.copy_(torch.tensor(lengths, dtype=torch.int32))
        eager = b.run()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kept, eager), i


@gpu
def test_refused_calls():
    b = _Batch([40, 3], 4, 2, 64, GgmlDType.Q8_0)
    c, q, t, n = b.cache, b.q, b.table, b.len
    for args in [(q.float(), t, n), (q[:1], t, n), (q[:, :3], t, n), (q[:, :0], t, n), (q[..., :32], t, n), (q.cpu(), t, n), (q[0], t, n),
                 (q, t.long(), n), (q, t[:1], n), (q, t[0], n), (q, t, n.long()), (q, t, n[:1]), (q, t.cpu(), n), (q, t, n.cpu()),
                 (q.clone().requires_grad_(True), t, n)]:
        with pytest.raises(ValueError):
            c.attend(*args)
    with pytest.raises(ValueError):
        c.attend(q, t, n, out=torch.empty(2, 4, 64, device="cuda"))
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(MoldqError):
            c.attend(q, t, n, scale=scale)
    assert c.attend(q[:0], t[:0], n[:0]).shape == (0, 4, 64)


def _cache(dtype=8, kv=2, dim=64, page=32, pages=3, data=4096):
    return _lib.KvCacheC(data, pages, dtype, kv, dim, page)


def test_argument_checks():
    lib = _lib.load()
    far = 1 << 40

    def call(c=None, q=4096, qs=(256, 64), batch=3, heads=4, table=4096, ts=4, pages=4, lengths=4096, scale=0.1, out=far, os=(256, 64),
             scratch=4096, size=1 << 30):
        c = c or _cache()
        return lib.mq_cache_attention(ctypes.byref(c), q, *qs, batch, heads, table, ts, pages, lengths, scale, out, *os, scratch, size, None)
    for kw in (dict(c=_cache(dtype=12)), dict(c=_cache(data=None)), dict(c=_cache(pages=0)), dict(c=_cache(data=4100)), dict(q=None), dict(q=4100),
               dict(qs=(252, 64)), dict(qs=(-256, 64)), dict(batch=-1), dict(heads=0), dict(heads=5), dict(table=None), dict(ts=3), dict(pages=-1),
               dict(pages=1 << 31, ts=1 << 31), dict(pages=1 << 26, ts=1 << 26), dict(lengths=None), dict(lengths=4098), dict(scale=0.0),
               dict(scale=float("nan")), dict(out=None), dict(out=4096 + 1024), dict(os=(128, 64)), dict(os=(256, 32)),
               dict(scratch=None, pages=64, ts=64), dict(size=100, pages=64, ts=64), dict(batch=1 << 30)):
        assert call(**kw) == -1, kw
    with pytest.raises(MoldqError):
        _lib.check(call(q=None))
    assert call(batch=0, q=None, lengths=None) == 0
    assert lib.mq_cache_attention(None, None, 0, 0, 0, 1, None, 0, 0, None, 1.0, None, 0, 0, None, 0, None) == -1
    size = lib.mq_cache_attention_scratch_size
    assert size(None, 1, 4, 4) == 0 and size(ctypes.byref(_cache()), 0, 4, 4) == 0 and size(ctypes.byref(_cache()), 1, 4, 64) > 0
    assert size(ctypes.byref(_cache()), 1, 4, 4) == 0      # a workgroup takes a whole head: no shares to join


@pytest.mark.skipif(HIPCC is None, reason="hipcc not available")
def test_kernels_do_not_spill(tmp_path):
    funcs = {k: v for k, v in _functions(_asm(tmp_path, "mq_decode.hip")).items() if "_kernel" in k}
    assert len(funcs) == 20
    for name, (_, meta) in funcs.items():
        assert meta.get("ScratchSize", 0) == 0, (name, meta)
