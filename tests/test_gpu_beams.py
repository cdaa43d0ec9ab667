"""Beam search's selection (select_beams) and reordering of cached sequences (BeamStates).

Selection is compared with float64 log_softmax of the same logits, sorted on the host: parents and
tokens exactly, totals within 2^-23 of their size (one rounding to f32 at half a step, 2^-24, and the
sum of exponentials: each off by 2^-23 of itself and, for its argument's rounding, by t 2^-23 where
it is 2^-t of the largest, together below 2^-22 of the sum, so 2^-22 absolute in its logarithm).
Random logits leave neighbouring totals of different beams further apart than that, which the
oracle checks before it compares."""
import ctypes
import random

import pytest

torch = pytest.importorskip("torch")

from mold_amd import GgmlDType, _lib
from mold_amd import text_attention as TA
from mold_amd.beams import BeamStates, select_beams

gpu = pytest.mark.gpu
BF = torch.bfloat16
INF, NAN = float("inf"), float("nan")


def _oracle(logits, scores, count, last=None, stop=None, apart=True):
    """Lists of (total, parent, token) of each request, by the definition, on the host."""
    out = []
    for i in range(logits.shape[0]):
        found = []
        for b in range(logits.shape[1]):
            score = float(scores[i, b])
            if abs(score) == INF or score != score:
                continue
            if stop is not None and int(last[i, b]) == stop:
                found.append((score, b, 0, stop))
                continue
            x = logits[i, b].double()
            if torch.isnan(x).any() or (x == INF).any() or (x == -INF).all():
                continue
            m = x.max()
            total = score + ((x - m) - (x - m).exp().sum().log())
            order = torch.sort(x, descending=True, stable=True).indices[:count]     # equal logits: the lower token first
            found += [(t, b, at, k) for at, (t, k) in enumerate(zip(total[order].tolist(), order.tolist())) if x[k] > -INF]
        found.sort(key=lambda f: (-f[0], f[1], f[2]))
        if apart:      # totals that lie closer than the bound may come in either order
            near = [p for p, q in zip(found[:count], found[1:count + 1]) if p[1] != q[1] and p[0] - q[0] < 2.0 ** -20 * max(1, abs(p[0]))]
            assert not near, "the oracle cannot tell: choose other inputs"
        out.append([(t, b, k) for t, b, _, k in found[:count]] + [(-INF, 0, -1)] * (count - len(found)))
    return out


def _check(logits, scores, count, last=None, stop=None, apart=True):
    totals, parents, tokens = select_beams(logits, scores, count, last, stop)
    assert totals.dtype == torch.float32 and parents.dtype == torch.int32 and tokens.dtype == torch.int64
    want = _oracle(logits, scores, count, last, stop, apart)
    assert parents.tolist() == [[b for _, b, _ in r] for r in want]
    assert tokens.tolist() == [[k for _, _, k in r] for r in want]
    for got, row in zip(totals.tolist(), want):
        for g, (t, _, _) in zip(got, row):
            assert g == t or abs(g - t) <= 2.0 ** -23 * abs(t) + 2.0 ** -22, (g, t)


def _logits(n, beams, vocab, dtype=torch.float32, seed=0, size=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed + vocab)
    x = torch.randn((n, beams, vocab), device="cuda", generator=g) * size
    return x.to(dtype), -5 * torch.rand((n, beams), device="cuda", generator=g)


@gpu
@pytest.mark.parametrize("vocab", [1, 2, 7, 63, 64, 65, 1000, 4097, 32001, 151111])
@pytest.mark.parametrize("dtype", [torch.float32, BF], ids=["f32", "bf16"])
def test_select(vocab, dtype):
    for n, beams, count in [(1, 1, 1), (1, 4, 4), (3, 5, 10), (2, 3, 64), (40, 2, 3)]:
        if vocab > 5000 and n * beams > 20:
            n = 5
        logits, scores = _logits(n, beams, vocab, dtype, seed=n)
        _check(logits, scores, count)


@gpu
def test_many_beams():
    for n, beams, count, vocab in [(1, 64, 64, 500), (2, 64, 1, 3), (3, 17, 33, 5000), (1, 64, 64, 1), (2, 8, 64, 4096), (2, 8, 64, 4097), (2, 7, 12, 900), (129, 2, 3, 40)]:
        logits, scores = _logits(n, beams, vocab, seed=9)
        _check(logits, scores, count)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, BF], ids=["f32", "bf16"])
@pytest.mark.parametrize("n,beams,count,vocab", [(255, 4, 3, 9001), (256, 4, 3, 9001), (301, 1, 2, 33333), (256, 2, 5, 20003), (260, 8, 1, 5003), (257, 5, 2, 7001)])
def test_many_requests(n, beams, count, vocab, dtype):
    """On both sides of where a workgroup reads a whole request."""
    logits, scores = _logits(n, beams, vocab, dtype, seed=n)
    _check(logits, scores, count)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, BF], ids=["f32", "bf16"])
def test_ties(dtype):
    """Equal logits in any number and place: the lowest tokens, of equal beams the lowest beam."""
    for vocab in (5, 64, 300, 9000):
        flat = torch.zeros((2, 3, vocab), dtype=dtype, device="cuda")
        for count in (1, 4, 20, 64):
            _check(flat, torch.zeros((2, 3), device="cuda"), count, apart=False)
        few = torch.randint(0, 4, (2, 3, vocab), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(dtype)
        few[:, 1] = few[:, 0]
        few[0, :, -1] = 9
        zeros = torch.where(torch.rand((2, 3, vocab), device="cuda") < 0.5, -0.0, 0.0).to(dtype)
        for x in (few, zeros):
            for count in (1, 7, 64):
                _check(x, torch.zeros((2, 3), device="cuda"), count, apart=False)


@gpu
@pytest.mark.parametrize("kind", ["rising", "falling", "steps", "one", "far"])
def test_orders(kind):
    """Logits whose order makes every one enter the list, or none after the first."""
    for vocab in (700, 40001):
        x = torch.linspace(-20, 20, vocab, device="cuda")
        x = {"rising": x, "falling": x.flip(0), "steps": x.view(-1)[torch.randperm(vocab, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))],
             "one": torch.where(torch.arange(vocab, device="cuda") == vocab - 2, 50.0, x * 0.01), "far": x * 1e30}[kind]
        scores = torch.tensor([[0.0, -0.37]], device="cuda")
        logits = torch.stack([x, x.roll(17)])[None].contiguous()
        _check(logits, scores, 9, apart=False) if kind == "far" else _check(logits, scores, 9)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, BF], ids=["f32", "bf16"])
def test_masks_and_what_is_not_a_number(dtype):
    least = torch.finfo(dtype).min
    for vocab in (50, 3001, 20000):
        logits, scores = _logits(9, 3, vocab, dtype, seed=4)
        logits[0, :, 5:] = -INF                              # five tokens each
        logits[1, 0] = -INF                                  # none
        logits[2, 1, vocab // 2] = NAN
        logits[3, 2, vocab - 1] = INF
        logits[4] = -INF
        logits[5, :, 1:] = least
        logits[6, 1] = least                                 # all alike
        logits[7, :, ::2] = -INF
        logits[8, 2, 0] = torch.finfo(dtype).max
        scores[7, 0], scores[7, 1], scores[8, 0] = -INF, NAN, INF
        for count in (3, 20):
            _check(logits, scores, count, apart=False)
    logits, scores = _logits(2, 4, 1000)                     # a search's first step: one beam that counts
    scores[:, 1:] = -INF
    _check(logits, scores, 4)


@gpu
@pytest.mark.parametrize("vocab", [5000, 20001])
def test_stopped_beams(vocab):
    logits, scores = _logits(6, 4, vocab, seed=5)
    scores[5] = -0.01
    last = torch.full((6, 4), 3, device="cuda")
    last[1, 2] = last[2, :3] = last[3] = last[4, 0] = last[5, 1] = 11
    logits[4, 0] = NAN                                       # an ended beam's logits are not looked at
    logits[3] = INF
    scores[2, 1] = -INF
    for count in (1, 4, 8):
        _check(logits, scores, count, last, 11)
    _check(logits, scores, 4, last, 4999)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, BF], ids=["f32", "bf16"])
def test_strides_and_alignment(dtype):
    """Rows that start anywhere, apart or one for all beams."""
    n, beams, vocab = 3, 4, 997
    wide = torch.randn((n, beams + 1, vocab + 6), device="cuda", generator=torch.Generator(device="cuda").manual_seed(6)).to(dtype) * 2
    scores = -torch.rand((n, beams), device="cuda") * 3
    for at in range(6):
        view = wide[:, 1:, at:at + vocab]
        got, want = select_beams(view, scores, 6), select_beams(view.contiguous(), scores, 6)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), at
        _check(view, scores, 6)
    by_token = wide[:, 1:, :vocab].transpose(1, 2).contiguous().transpose(1, 2)
    assert all(torch.equal(a, b) for a, b in zip(select_beams(by_token, scores, 6), select_beams(wide[:, 1:, :vocab], scores, 6)))
    same = wide[:, :1, :vocab].expand(n, beams, vocab)
    assert all(torch.equal(a, b) for a, b in zip(select_beams(same, scores, 6), select_beams(same.contiguous(), scores, 6)))
    pairs = torch.stack([scores, scores], 2)[..., 1]
    assert all(torch.equal(a, b) for a, b in zip(select_beams(same, pairs, 6), select_beams(same, scores, 6)))


@gpu
def test_the_runs_of_a_row_do_not_matter():
    """A request alone, whose rows are cut into many runs, and among others: the same beams and tokens."""
    logits, scores = _logits(60, 4, 60000, seed=8)
    every = select_beams(logits, scores, 8)
    for i in (0, 31, 59):
        alone = select_beams(logits[i:i + 1], scores[i:i + 1], 8)
        assert torch.equal(alone[1], every[1][i:i + 1]) and torch.equal(alone[2], every[2][i:i + 1])
        torch.testing.assert_close(alone[0], every[0][i:i + 1], rtol=2.0 ** -23, atol=2.0 ** -22)


@gpu
def test_no_requests_and_refusals():
    logits, scores = _logits(2, 3, 100)
    last = torch.zeros((2, 3), dtype=torch.int64, device="cuda")
    assert [x.shape for x in select_beams(logits[:0], scores[:0], 5)] == [(0, 5)] * 3
    for args, kw in (((logits.half(), scores), {}), ((logits[0], scores), {}), ((logits.cpu(), scores), {}), ((logits, scores.double()), {}), ((logits, scores[:1]), {}),
                     ((logits, scores.cpu()), {}), ((logits, scores, 0), {}), ((logits, scores, 65), {}), ((logits[:, :0], scores[:, :0]), {}), ((logits[..., :0], scores), {}),
                     ((logits, scores), {"last": last}), ((logits, scores), {"stop": 3}), ((logits, scores), {"last": last, "stop": 100}), ((logits, scores), {"last": last, "stop": -1}),
                     ((logits, scores), {"last": last.int(), "stop": 1}), ((logits, scores), {"last": last[:1], "stop": 1}), ((logits.clone().requires_grad_(), scores), {}),
                     ((logits.expand(2, 3, 100).repeat(1, 22, 1), scores.repeat(1, 22)), {})):
        with pytest.raises(ValueError):
            select_beams(*args, **kw)


# ------------------------------------------------------------------ reordering

def _states(layers, pages, kv, dim, page, t, seed=0):
    caches = [TA.KvCache(pages, kv, dim, page_tokens=page, dtype=t) for _ in range(layers)]
    for i, c in enumerate(caches):
        c.data.copy_(torch.randint(0, 256, c.data.shape, dtype=torch.uint8, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed + i)))
    return caches


def _raw(cache):
    """The cache's bytes on the host, as [pages, heads, tiles, ..]."""
    return cache.data.view(cache.pages, cache.kv_heads, cache.page_tokens // 32, -1).cpu()


def _bytes_of(cache, pages, length, data=None):
    """What a sequence of `length` tokens over `pages` holds: the raw tiles that its tokens reach, as [heads, tiles, ..] of each page."""
    data, out = _raw(cache) if data is None else data, []
    for c, page in enumerate(pages):
        left = min(cache.page_tokens, length - c * cache.page_tokens)
        if left <= 0:
            break
        out.append(data[page, :, :-(-left // 32)].clone())
    return out


def _tables(n, beams, width, lengths, page, rng):
    """A table as a search has it: shared whole pages, then pages of each row's own; and how many pages there are."""
    table, at = [], 0
    for i in range(n):
        full = lengths[i] // page
        common = list(range(at, at + full))
        at += full
        for _ in range(beams):
            own = list(range(at, at + width - full))
            at += len(own)
            table.append(common[:width] + own)
    order = list(range(at))
    rng.shuffle(order)
    return [[order[p] for p in row] for row in table], at


@gpu
@pytest.mark.parametrize("t", [GgmlDType.BF16, GgmlDType.Q8_0, GgmlDType.Q4_0], ids=lambda t: t.name)
@pytest.mark.parametrize("beams", [2, 3, 8, 64])
def test_reorder(t, beams):
    """After it each row holds what its parent held; from the partial page on no two rows share a
    page; pages that no row had there keep their bytes; several steps one after another."""
    rng = random.Random(beams)
    for n, kv, dim, page, layers in [(1, 1, 64, 32, 1), (4, 3, 128, 96, 2), (3, 2, 64, 256, 3)]:
        if beams == 64 and n > 1:
            n = 2
        lengths = [rng.choice([0, 1, 31, 32, 33, page - 1, page, page + 1, 2 * page - 7]) for _ in range(n)]
        width = 2 * page // page + 2
        table, pages = _tables(n, beams, width, lengths, page, rng)
        caches = _states(layers, pages + 2, kv, dim, page, t)
        states, dev = BeamStates(caches), torch.tensor(table, dtype=torch.int32, device="cuda")
        now = torch.tensor([x for x in lengths for _ in range(beams)], dtype=torch.int32, device="cuda")
        for step in range(3):
            parents = [[rng.choice([j, 0, rng.randrange(beams), rng.randrange(beams)]) for j in range(beams)] for _ in range(n)]
            if step == 1:
                parents[0] = [beams - 1 - j for j in range(beams)]            # nothing but a permutation
            raw = [_raw(c) for c in caches]
            before = [[_bytes_of(c, table[i * beams + j], lengths[i], r) for j in range(beams)] for c, r in zip(caches, raw) for i in range(n)]
            states.reorder(dev, now, torch.tensor(parents, dtype=torch.int32, device="cuda"))
            after, now_raw = dev.tolist(), [_raw(c) for c in caches]
            for i in range(n):
                full = lengths[i] // page
                rows = after[i * beams:(i + 1) * beams]
                own = [p for r in rows for p in r[full:]]
                assert len(set(own)) == len(own)
                assert sorted(own) == sorted(p for r in table[i * beams:(i + 1) * beams] for p in r[full:])
                for j, r in enumerate(rows):
                    assert r[:full] == table[i * beams + parents[i][j]][:full]
                    for layer, c in enumerate(caches):
                        got = _bytes_of(c, r, lengths[i], now_raw[layer])
                        assert len(got) == len(before[layer * n + i][parents[i][j]])
                        assert all(torch.equal(a, b) for a, b in zip(got, before[layer * n + i][parents[i][j]])), (i, j, layer)
                kept = set(parents[i])
                copies = beams - len(kept) if lengths[i] % page else 0
                changed = sum(not torch.equal(now_raw[0][p], raw[0][p]) for p in {p for r in rows for p in r[full:full + 1]})
                assert changed <= copies
            table = after


@gpu
def test_reorder_of_what_is_no_beam_and_past_the_table():
    rng = random.Random(1)
    table, pages = _tables(3, 4, 3, [40, 96, 200], 32, rng)          # the third longer than its table
    table[0][1] = -1                                          # a partial page that is none of the cache's
    caches = _states(2, pages, 2, 64, 32, GgmlDType.Q8_0)
    held = [c.data.clone() for c in caches]
    dev, lengths = torch.tensor(table, dtype=torch.int32, device="cuda"), torch.tensor([40, 96, 200], dtype=torch.int32, device="cuda").repeat_interleave(4)
    BeamStates(caches).reorder(dev, lengths, torch.tensor([[0, -1, 4, 99], [-5, 1, 2, 3], [7, 1, 2, 3]], dtype=torch.int32, device="cuda"))
    assert dev.tolist() == table and all(torch.equal(c.data, h) for c, h in zip(caches, held))
    BeamStates(caches).reorder(dev, lengths, torch.tensor([[0, 0, 2, 3], [1, 1, 1, 1], [3, 3, 3, 3]], dtype=torch.int32, device="cuda"))
    assert all(torch.equal(c.data, h) for c, h in zip(caches, held))
    got = dev.tolist()
    assert got[4:8] == [table[5]] * 4 and got[8:] == [table[11]] * 4
    negative = torch.full((12,), -7, dtype=torch.int32, device="cuda")
    BeamStates(caches).reorder(dev, negative, torch.tensor([[1, 1, 1, 1]] * 3, dtype=torch.int32, device="cuda"))
    assert dev.tolist() == got


@gpu
def test_reorder_many_layers_and_views():
    """More caches than one launch takes, a table that is a view, lengths and parents that are too."""
    rng = random.Random(2)
    table, pages = _tables(2, 3, 2, [20, 45], 32, rng)
    caches = _states(67, pages, 1, 64, 32, GgmlDType.Q4_0)
    wide = torch.full((6, 5), 77, dtype=torch.int32, device="cuda")
    wide[:, 2:4] = torch.tensor(table, dtype=torch.int32, device="cuda")
    lengths = torch.tensor([20] * 3 + [45] * 3, dtype=torch.int32, device="cuda")
    parents = torch.tensor([[1, 1, 0], [2, 2, 2]], dtype=torch.int32, device="cuda")
    want = [[_bytes_of(c, table[3 * i + int(parents[i, j])], [20, 45][i]) for i in range(2) for j in range(3)] for c in caches]
    BeamStates(caches).reorder(wide[:, 2:4], torch.stack([lengths, lengths], 1)[:, 0], torch.stack([parents, parents], 2)[..., 1])
    assert (wide[:, [0, 1, 4]] == 77).all()
    after = wide[:, 2:4].tolist()
    for c, w in zip(caches, want):
        for row, (pages_of, expect) in enumerate(zip(after, w)):
            assert all(torch.equal(a, b) for a, b in zip(_bytes_of(c, pages_of, [20, 45][row // 3]), expect))


@gpu
def test_reorder_of_many_requests():
    """More requests than one launch copies for, most of them without copies, the last with some."""
    n, beams, page = 2500, 2, 32
    table = torch.arange(n * beams * 2, dtype=torch.int32, device="cuda").view(n * beams, 2)
    cache = _states(1, n * beams * 2, 1, 64, page, GgmlDType.Q4_0)[0]
    parents = torch.tensor([[0, 1]] * n, dtype=torch.int32, device="cuda")
    some = [0, 63, 64, 700, 1023, 1024, 1025, 2047, 2048, 2499]
    parents[some] = torch.tensor([1, 1], dtype=torch.int32, device="cuda")
    lengths = torch.full((n * beams,), 7, dtype=torch.int32, device="cuda")
    want = _raw(cache)
    for i in some:
        want[4 * i] = want[4 * i + 2]
    BeamStates([cache]).reorder(table, lengths, parents)
    assert torch.equal(_raw(cache), want)
    assert torch.equal(table, torch.arange(n * beams * 2, dtype=torch.int32, device="cuda").view(n * beams, 2))


@gpu
def test_states_dropped_behind_another_stream():
    """The caches' memory is not given to other tensors before a reordering that still uses it has ended."""
    from tests.test_gpu_text_streams import _dropped_on
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(4, 2)
    lengths, parents = torch.full((4,), 7, dtype=torch.int32, device="cuda"), torch.tensor([[1, 1, 3, 3]], dtype=torch.int32, device="cuda")
    caches = _states(1, 8, 1, 64, 32, GgmlDType.Q8_0)
    states = BeamStates(caches)
    torch.cuda.synchronize()

    def own():
        nonlocal caches, states
        at = caches[0].data.data_ptr(), caches[0].data.numel()
        caches = states = None
        return at
    _, early = _dropped_on(torch.cuda.Stream(), lambda: states.reorder(table, lengths, parents), own)
    assert not early


@gpu
def test_two_streams_at_once():
    """Selections and reorderings of different sizes on two streams, neither waiting for the other."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    jobs = []
    for i, (n, beams, vocab, count) in enumerate([(5, 4, 40001, 4), (40, 3, 20000, 3)]):
        logits, scores = _logits(n, beams, vocab, seed=30 + i)
        table = torch.arange(n * beams * 2, dtype=torch.int32, device="cuda").view(n * beams, 2)
        caches = _states(3, n * beams * 2, 2, 64, 32, GgmlDType.Q8_0, seed=i)
        jobs.append((logits, scores, count, BeamStates(caches), table, torch.full((n * beams,), 9, dtype=torch.int32, device="cuda"), caches))

    def run(job, times):
        out = []
        for _ in range(times):
            got = select_beams(job[0], job[1], job[2])
            job[3].reorder(job[4], job[5], got[1])
            out.append(got)
        return out
    start = [(j[4].clone(), [c.data.clone() for c in j[6]]) for j in jobs]
    want = [(run(j, 20), j[4].clone(), [c.data.clone() for c in j[6]]) for j in jobs]
    for j, (table, data) in zip(jobs, start):
        j[4].copy_(table)
        for c, d in zip(j[6], data):
            c.data.copy_(d)
    torch.cuda.synchronize()
    got = []
    for j, s in zip(jobs, streams):
        with torch.cuda.stream(s):
            got.append(run(j, 20))
    torch.cuda.synchronize()
    for j, g, (w, table, data) in zip(jobs, got, want):
        assert all(torch.equal(a, b) for x, y in zip(g, w) for a, b in zip(x, y))
        assert torch.equal(j[4], table) and all(torch.equal(c.data, d) for c, d in zip(j[6], data))


@gpu
def test_reorder_refusals():
    caches = _states(2, 8, 1, 64, 32, GgmlDType.Q8_0)
    states = BeamStates(caches)
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(4, 2)
    lengths, parents = torch.full((4,), 5, dtype=torch.int32, device="cuda"), torch.zeros((2, 2), dtype=torch.int32, device="cuda")
    for args in ((table.long(), lengths, parents), (table[:3], lengths, parents), (table.cpu(), lengths, parents), (table, lengths.long(), parents), (table, lengths[:3], parents),
                 (table, lengths, parents.long()), (table, lengths, parents.view(-1)), (table, lengths, parents[:, :0]), (table.t().contiguous().t(), lengths, parents),
                 (table[:1].expand(4, 2), lengths, parents), (table, lengths, torch.zeros((1, 65), dtype=torch.int32, device="cuda"))):
        with pytest.raises(ValueError):
            states.reorder(*args)
    for bad in ([], [caches[0], caches[0]], [caches[0], TA.KvCache(8, 2, 64, page_tokens=32)], [caches[0], TA.KvCache(9, 1, 64, page_tokens=32)]):
        with pytest.raises(ValueError):
            BeamStates(bad)
    states.reorder(table[:0], lengths[:0], parents[:0])
    one = table.clone()
    states.reorder(one, lengths, torch.zeros((4, 1), dtype=torch.int32, device="cuda"))
    assert torch.equal(one, table)


@gpu
@pytest.mark.parametrize("vocab", [3001, 40001])
def test_captured(vocab):
    """A step's selection and reordering, replayed: each replay goes on from the one before."""
    rng = random.Random(4)
    table, pages = _tables(2, 4, 3, [40, 40], 32, rng)
    logits, scores = _logits(2, 4, vocab, seed=3)
    lengths = torch.full((8,), 40, dtype=torch.int32, device="cuda")
    graphed, eager = (_states(2, pages, 2, 64, 32, GgmlDType.Q8_0) for _ in range(2))
    a, b = (torch.tensor(table, dtype=torch.int32, device="cuda") for _ in range(2))
    sa, sb, s = BeamStates(graphed), BeamStates(eager), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        _, p, _ = select_beams(logits, scores)
        sa.reorder(a, lengths, p)
        with torch.cuda.graph(graph, stream=s):
            out = select_beams(logits, scores)
            sa.reorder(a, lengths, out[1])
    torch.cuda.current_stream().wait_stream(s)
    sb.reorder(b, lengths, select_beams(logits, scores)[1])
    for i in range(4):
        x = _logits(2, 4, vocab, seed=20 + i)
        logits.copy_(x[0]), scores.copy_(x[1])
        want = select_beams(logits, scores)
        sb.reorder(b, lengths, want[1])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want)), i
        assert torch.equal(a, b) and all(torch.equal(x.data, y.data) for x, y in zip(graphed, eager)), i


def test_refusals_of_the_library():
    """On the CPU: every fault is found before anything is launched."""
    lib, a, bad = _lib.load(), 4096, _lib.MQ_E_INVALID
    need = lib.mq_beam_select_scratch_size(3, 4, 100000, 4, 0)
    assert need > 0 and lib.mq_beam_select_scratch_size(0, 4, 100000, 4, 0) == 0 and lib.mq_beam_select_scratch_size(3, 4, 1000, 4, 30) == 0
    for args in ((-1, 4, 100000, 4), (3, 0, 100000, 4), (3, 65, 100000, 4), (3, 4, 0, 4), (3, 4, 1 << 31, 4), (3, 4, 100000, 0), (3, 4, 100000, 65), ((1 << 20) + 1, 4, 100000, 4)):
        assert lib.mq_beam_select_scratch_size(*args, 0) == 0, args
    assert lib.mq_beam_select_scratch_size(3, 4, 100000, 4, 1) == 0
    ok = dict(logits=a, dtype=0, n=3, beams=4, vocab=100000, rs=400000, bs=100000, scores=a, last=a, stop=7, count=4, totals=a, parents=a, tokens=a, scratch=a, size=need, stream=None)
    for change in (dict(logits=None), dict(dtype=1), dict(n=-1), dict(n=(1 << 20) + 1), dict(beams=0), dict(beams=65), dict(vocab=0), dict(vocab=1 << 31), dict(rs=-1),
                   dict(bs=1 << 40), dict(scores=None), dict(stop=-1), dict(stop=100000), dict(count=0), dict(count=65), dict(totals=None), dict(parents=None),
                   dict(tokens=None), dict(scratch=None), dict(size=need - 1), dict(logits=a + 2), dict(logits=a + 1, dtype=30), dict(scores=a + 2), dict(last=a + 4),
                   dict(totals=a + 1), dict(parents=a + 2), dict(tokens=a + 4), dict(scratch=a + 8), dict(n=1 << 20, beams=64, size=1 << 60)):
        assert lib.mq_beam_select(*{**ok, **change}.values()) == bad, change
    assert lib.mq_beam_select(*{**ok, "n": 0}.values()) == 0
    assert lib.mq_beam_reorder_scratch_size(2, 4) > 0
    for args in ((-1, 4), (2, 0), (2, 65), ((1 << 20) + 1, 2)):
        assert lib.mq_beam_reorder_scratch_size(*args) == 0
    two = (_lib.KvCacheC * 2)(_lib.KvCacheC(a, 4, 8, 2, 128, 64), _lib.KvCacheC(a, 4, 8, 2, 128, 64))
    ok = dict(caches=two, count=2, table=a, stride=5, width=5, lengths=a, parents=a, n=2, beams=4, scratch=a, size=lib.mq_beam_reorder_scratch_size(2, 4), stream=None)
    for change in (dict(caches=None), dict(count=0), dict(count=257), dict(table=None), dict(stride=4), dict(stride=1 << 40), dict(width=-1), dict(width=1 << 31), dict(lengths=None), dict(parents=None),
                   dict(n=-1), dict(n=(1 << 20) + 1), dict(beams=0), dict(beams=65), dict(scratch=None), dict(size=1), dict(table=a + 2), dict(lengths=a + 1), dict(parents=a + 2), dict(scratch=a + 8)):
        assert lib.mq_beam_reorder(*{**ok, **change}.values()) == bad, change
    assert lib.mq_beam_reorder(*{**ok, "n": 0}.values()) == 0 and lib.mq_beam_reorder(*{**ok, "beams": 1}.values()) == 0
    for field, value in (("data", None), ("data", a + 4), ("pages", 5), ("dtype", 30), ("kv_heads", 1), ("head_dim", 64), ("page_tokens", 32), ("page_tokens", 31)):
        other = (_lib.KvCacheC * 2)(two[0], two[1])
        setattr(other[1], field, value)
        assert lib.mq_beam_reorder(*{**ok, "caches": other}.values()) == bad, field
