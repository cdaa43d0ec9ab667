"""mq_prompt_attention against float64 attention: the edges of its key halves (32), key blocks
(64) and token tiles (32 to 128 by the heads' groups), packed prompts, views, what a row must
not see, and its refusals.

The bound on the relative error is that of the roundings to bf16: of the probabilities and of
the output, 1.66e-3 each on average (2^-9 / sqrt(3) relative to the mantissa's lower end, uniform
mantissas), 2.4e-3 together; 3e-3 is asserted over a whole output."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from mold_amd import MoldqError, _lib
from mold_amd import text_attention as TA
from tests.test_build_checks import HIPCC, _asm, _functions, _m0_outside_asm

gpu = pytest.mark.gpu
BOUND = 3e-3
BF = torch.bfloat16


def _inputs(lengths, heads, kv, dim, seed=0, sharp=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + 7919 * sum(lengths) + dim + heads)
    x = torch.randn((sum(lengths), heads + 2 * kv, dim), device="cuda", generator=g)
    x[:, :heads] *= sharp
    x = x.to(BF)
    return x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]


def _ref(q, k, v, lengths, scale=None):
    q, k, v = (t.double().cpu() for t in (q, k, v))
    group, scale = q.shape[1] // k.shape[1], q.shape[2] ** -0.5 if scale is None else scale
    out, at = torch.empty_like(q), 0
    for n in lengths:
        r = slice(at, at + n)
        kk, vv = (t[r].repeat_interleave(group, 1).transpose(0, 1) for t in (k, v))
        s = q[r].transpose(0, 1) @ kk.transpose(1, 2) * scale
        s = s.masked_fill(torch.ones(n, n, dtype=torch.bool).triu(1), float("-inf"))
        out[r] = (torch.softmax(s, -1) @ vv).transpose(0, 1)
        at += n
    return out


def _err(out, ref):
    return ((out.double().cpu() - ref).norm() / ref.norm()).item()


def _run(q, k, v, lengths, **kw):
    return TA.prompt_attention(q, k, v, TA.PromptPlan(lengths, q.shape[1], k.shape[1], q.shape[2]), **kw)


def _run_whole(q, k, v, lengths):
    """The same rows in a batch of so many tiles that each takes all its keys in one part, before
    many prompts of zeros."""
    more = [1000] * 120
    pad = lambda t: torch.cat([t, torch.zeros((sum(more),) + t.shape[1:], dtype=t.dtype, device="cuda")])
    plan = TA.PromptPlan(lengths + more, q.shape[1], k.shape[1], q.shape[2])
    assert plan.c.parts == 1 and TA.PromptPlan(lengths, q.shape[1], k.shape[1], q.shape[2]).c.parts == 2
    return TA.prompt_attention(pad(q), pad(k), pad(v), plan)[:q.shape[0]]


@gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 2), (8, 2), (7, 1), (6, 2), (16, 1), (12, 12)])
def test_lengths_and_groups(heads, kv, dim):
    for n in (1, 2, 31, 32, 33, 63, 64, 65, 95, 96, 97, 127, 128, 129, 160, 193, 257, 320, 577):
        q, k, v = _inputs([n], heads, kv, dim)
        ref = _ref(q, k, v, [n])
        assert _err(_run(q, k, v, [n]), ref) < BOUND, n
        if n in (1, 31, 33, 64, 96, 129, 257, 577):
            assert _err(_run_whole(q, k, v, [n]), ref) < BOUND, n


@gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv", [(2, 2), (4, 2), (8, 2), (8, 1)])
def test_packed_prompts(heads, kv, dim):
    """Prompts of no, one and many tokens beside each other, in any order; each as if it were alone."""
    lengths = [3, 0, 1, 130, 64, 0, 33, 257, 1, 31, 0]
    q, k, v = _inputs(lengths, heads, kv, dim)
    out = _run(q, k, v, lengths)
    ref = _ref(q, k, v, lengths)
    assert _err(out, ref) < BOUND and _err(_run_whole(q, k, v, lengths), ref) < BOUND
    at = 0
    for n in lengths:
        if n:
            alone = _run(q[at:at + n], k[at:at + n], v[at:at + n], [n])
            assert torch.equal(alone, out[at:at + n]), n
        at += n


@gpu
@pytest.mark.parametrize("lengths", [[], [0], [0, 0, 0]])
def test_no_tokens(lengths):
    q = torch.empty((0, 4, 64), dtype=BF, device="cuda")
    assert _run(q, q[:, :2], q[:, :2], lengths).shape == (0, 4, 64)


@gpu
@pytest.mark.parametrize("sharp,scale", [(0.0, None), (30.0, None), (1.0, 0.5), (1.0, 1e-4)])
def test_flat_and_one_hot_rows(sharp, scale):
    lengths = [200, 77]
    q, k, v = _inputs(lengths, 4, 2, 128, seed=5, sharp=sharp)
    assert _err(_run(q, k, v, lengths, scale=scale), _ref(q, k, v, lengths, scale)) < BOUND


@gpu
@pytest.mark.parametrize("run", [_run, _run_whole], ids=["parts", "whole"])
@pytest.mark.parametrize("step", [0.01, 0.2, 0.3, 5.0, -0.2])
@pytest.mark.parametrize("dim", [64, 128])
def test_rising_scores(dim, step, run):
    """Scores that rise or fall from key to key by a little or by much, to maxima that differ by row and head."""
    n = 700
    q, k, v = (t.clone() for t in _inputs([n], 4, 2, dim))
    at = torch.arange(n, device="cuda", dtype=torch.float32)
    q[:, :, 0] = torch.tensor([1.0, 2.0, 4.0, 0.5], device="cuda", dtype=BF)
    k[:, :, 0] = (at * step * dim ** 0.5)[:, None].to(BF)
    k[:, :, 1] = (at % 7 * step * dim ** 0.5)[:, None].to(BF)
    assert _err(run(q, k, v, [n]), _ref(q, k, v, [n])) < BOUND


@gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("run", [_run, _run_whole], ids=["parts", "whole"])
def test_unseen_keys_do_not_reach_a_row(run, which, bad, dim):
    """A non-finite key or value of a later token, or of another prompt, changes no bit of a row;
    rows that see it become what the sum says."""
    lengths = [70, 100, 40]
    q, k, v = _inputs(lengths, 4, 2, dim, seed=9)
    clean = run(q, k, v, lengths)
    for at in (0, 31, 32, 50, 63, 64, 90, 99):
        k2, v2 = k.clone(), v.clone()
        (k2 if which == "k" else v2)[70 + at, 1, 5] = bad
        out = run(q, k2, v2, lengths)
        same = torch.cat([out[:70 + at], out[170:]])
        assert torch.equal(same, torch.cat([clean[:70 + at], clean[170:]])), at
        assert torch.equal(out[:, :2], clean[:, :2]), at           # the other group of heads
        hit = out[70 + at:170, 2:]
        if which == "v":
            assert torch.equal(torch.isnan(hit[:, :, 5]), torch.full_like(hit[:, :, 5], bad != bad, dtype=torch.bool)), at
            assert not torch.isfinite(hit[:, :, 5]).any(), at
            rest = [c for c in range(dim) if c != 5]
            assert torch.equal(hit[:, :, rest], clean[70 + at:170, 2:][:, :, rest]), at
        elif bad != bad:
            assert torch.isnan(hit).all(), at


@gpu
def test_infinities_of_both_signs_in_one_diagonal():
    """Rows that see +inf, then also -inf, of one value column: inf, then NaN."""
    q, k, v = _inputs([32], 2, 1, 64, seed=3)
    v = v.clone()
    v[10, 0, 7], v[20, 0, 7] = float("inf"), float("-inf")
    col = _run(q, k, v, [32])[:, 0, 7].float()
    assert torch.isfinite(col[:10]).all() and (col[10:20] == float("inf")).all() and torch.isnan(col[20:]).all()


@gpu
def test_views_and_strided_out():
    lengths = [65, 30]
    q, k, v = _inputs(lengths, 8, 2, 64, seed=11)
    want = _run(q.contiguous(), k.contiguous(), v.contiguous(), lengths)
    assert torch.equal(_run(q, k, v, lengths), want)
    heads_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    assert torch.equal(_run(*heads_first, lengths), want)
    odd = [torch.nn.functional.pad(t, (1, 2))[:, :, 1:65] for t in (q, k, v)]          # rows off 16 bytes: copied
    assert torch.equal(_run(*odd, lengths), want)
    assert torch.equal(_run(q, k[:, :1].expand(-1, 2, -1), v, lengths)[:, :4], want[:, :4])    # one k head for both groups
    for shape, cut in [((95, 10, 72), (slice(None), slice(1, 9), slice(0, 64))), ((95, 8, 67), (slice(None), slice(None), slice(2, 66)))]:
        buf = torch.full(shape, 3.0, dtype=BF, device="cuda")
        view = buf[cut]
        assert _run(q, k, v, lengths, out=view) is view and torch.equal(view, want)
        view.fill_(3.0)
        assert bool((buf == 3.0).all())
    buf = torch.full((8, 95, 64), 3.0, dtype=BF, device="cuda").transpose(0, 1)         # head-major out
    assert torch.equal(_run(q, k, v, lengths, out=buf), want)
    x = torch.cat([q, k, v], 1)
    assert torch.equal(_run(x[:, :8], x[:, 8:10], x[:, 10:], lengths, out=x[:, :8]), want)     # over q: through a temporary
    assert torch.equal(x[:, 8:10], k)
    host = torch.empty((95, 8, 64), dtype=BF)
    assert torch.equal(_run(q, k, v, lengths, out=host), want.cpu())


@gpu
def test_offsets_past_32_bits():
    """Rows 2^23 elements apart: 300 of them span 5 GB."""
    n, stride = 300, 1 << 23
    q, k, v = _inputs([n], 2, 1, 64, seed=2)
    want = _run(q, k, v, [n])
    big = torch.empty((n - 1) * stride + 256, dtype=BF, device="cuda")
    far = big.as_strided((n, 4, 64), (stride, 64, 1))
    far.copy_(torch.cat([q, k, v], 1))
    assert torch.equal(_run(far[:, :2], far[:, 2:3], far[:, 3:], [n]), want)
    assert torch.equal(_run(q, k, v, [n], out=far[:, :2]), want)


@gpu
def test_long_prompt_rows():
    """Sampled rows of a prompt whose tiles fill the chip several times."""
    n = 7001
    q, k, v = _inputs([n], 8, 2, 128, seed=4)
    out = _run(q, k, v, [n])
    assert TA.PromptPlan([n], 8, 2, 128).c.parts == 1
    for i in (0, 1, 2047, 2048, 4095, 6999, 7000):
        kk, vv = (t[:i + 1].double().repeat_interleave(4, 1).transpose(0, 1) for t in (k, v))
        w = torch.softmax((kk @ q[i].double().unsqueeze(2)).squeeze(2) / 128 ** 0.5, -1)
        ref = (w.unsqueeze(1) @ vv.contiguous()).squeeze(1)
        assert ((out[i].double() - ref).norm() / ref.norm()).item() < 1.5 * BOUND, i    # one row: 1024 values
    assert torch.equal(out, _run(q, k, v, [n]))


@gpu
def test_other_streams_and_graphs():
    lengths = [130, 45]
    q, k, v = _inputs(lengths, 8, 2, 128, seed=6)
    plan = TA.PromptPlan(lengths, 8, 2, 128)
    want = TA.prompt_attention(q, k, v, plan)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = TA.prompt_attention(q, k, v, plan)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            kept = TA.prompt_attention(q, k, v, plan)
    s.synchronize()
    assert torch.equal(got, want)
    for i in range(4):
        q.copy_(torch.randn_like(q))
        eager = TA.prompt_attention(q, k, v, plan)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kept, eager), i


@gpu
def test_refused_calls():
    q, k, v = _inputs([40], 4, 2, 64)
    plan = TA.PromptPlan([40], 4, 2, 64)
    bad = [(q.float(), k, v), (q, k, v[:39]), (q[:, :2], k, v), (q, k[:, :1], v), (q, k, v[..., :32]), (q.cpu(), k, v), (q, k, v[None])]
    for args in bad:
        with pytest.raises(ValueError):
            TA.prompt_attention(*args, plan)
    with pytest.raises(ValueError):
        TA.prompt_attention(q[:39], k[:39], v[:39], plan)
    with pytest.raises(ValueError):
        TA.prompt_attention(q.clone().requires_grad_(True), k, v, plan)
    with pytest.raises(ValueError):
        TA.prompt_attention(q, k, v, plan, out=torch.empty(40, 4, 64, device="cuda"))
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(MoldqError):
            TA.prompt_attention(q, k, v, plan, scale=scale)


def _plan(lengths, heads=4, kv=2, dim=64, capacity=64):
    lib, c = _lib.load(), _lib.PromptPlanC()
    tiles = (ctypes.c_int32 * (4 * max(1, capacity)))()
    rc = lib.mq_prompt_plan_make((ctypes.c_int64 * max(1, len(lengths)))(*lengths), len(lengths), heads, kv, dim, ctypes.byref(c),
                                 tiles if capacity else None, capacity)
    return rc, c, [tuple(tiles[4 * i:4 * i + 4]) for i in range(min(capacity, max(0, c.tiles)))]


@pytest.mark.parametrize("heads,kv,whole,split", [(4, 4, 128, 64), (4, 2, 64, 32), (8, 2, 32, 32), (7, 1, 128, 64), (6, 1, 64, 32), (12, 1, 32, 32)])
@pytest.mark.parametrize("parts", [1, 2])
def test_plan_covers_every_token_once(heads, kv, whole, split, parts):
    """Few tiles are split over the keys too (two parts), many are not."""
    lengths = [0, 5, 128, 129, 0, 64, 1, 300] + [50000] * (2 - parts) * 16
    rc, c, tiles = _plan(lengths, heads, kv, capacity=40000)
    tile = whole if parts == 1 else split
    assert rc == 0 and c.parts == parts
    assert c.tokens == sum(lengths) and c.tile_tokens == tile and c.tiles == sum(-(-n // tile) for n in lengths)
    starts = {}
    for start, n, first, _ in tiles[:c.tiles]:
        starts.setdefault((start, n), []).append(first)
    at, want = 0, {}
    for n in lengths:
        if n:
            want[(at, n)] = list(range(0, n, tile))
        at += n
    assert {key: sorted(f) for key, f in starts.items()} == want
    assert [t[2] for t in tiles[:c.tiles]] == sorted((t[2] for t in tiles[:c.tiles]), reverse=True)     # longest first


def test_plan_pairs_long_tiles_with_short_ones():
    """Where all workgroups run at once, those after a CU's first come from the short end."""
    rc, c, tiles = _plan([2000], 32, 8, 128)
    firsts = [t[2] // 32 for t in tiles[:c.tiles]]
    assert rc == 0 and c.parts == 1 and firsts == list(range(62, 30, -1)) + list(range(0, 31))


def test_argument_checks():
    lib = _lib.load()
    for kw in (dict(lengths=[-1]), dict(lengths=[1 << 31]), dict(lengths=[1 << 30, 1 << 30]), dict(dim=96), dict(heads=0), dict(kv=0),
               dict(heads=5), dict(lengths=[9000], capacity=10)):
        assert _plan(**{"lengths": [40], **kw})[0] == -1, kw
    assert lib.mq_prompt_plan_make(None, 1, 4, 2, 64, ctypes.byref(_lib.PromptPlanC()), None, 0) == -1
    assert lib.mq_prompt_plan_make(None, 0, 4, 2, 64, None, None, 0) == -1
    _, plan, _ = _plan([40])
    far = 1 << 40

    def call(plan=plan, tiles=4096, q=4096, qs=(256, 64), k=4096, ks=(128, 64), v=4096, vs=(128, 64), scale=0.1, out=far, os=(256, 64)):
        return lib.mq_prompt_attention(plan, tiles, q, *qs, k, *ks, v, *vs, scale, out, *os, None)
    foreign = _lib.PromptPlanC(40, 3, 4, 2, 64, 128, 1)
    bad = [dict(plan=None), dict(plan=foreign), dict(q=None), dict(tiles=None), dict(q=4100), dict(out=far + 2), dict(qs=(252, 64)),
           dict(ks=(-128, 64)), dict(vs=(1 << 24, 64)), dict(os=(128, 64)), dict(os=(256, 32)), dict(os=(0, 64)), dict(os=(64, 64 * 39)),
           dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(out=4096), dict(out=4096 + 2 * 128 * 39)]
    for kw in bad:
        assert call(**kw) == -1, kw
    with pytest.raises(MoldqError):
        _lib.check(call(q=None))
    empty = _plan([0, 0])[1]
    assert call(plan=empty, q=None, tiles=None) == 0


@pytest.mark.skipif(HIPCC is None, reason="hipcc not available")
def test_kernel_leaves_m0_alone_and_does_not_spill(tmp_path):
    funcs = {k: v for k, v in _functions(_asm(tmp_path, "mq_prompt.hip")).items() if "prompt_kernel" in k}
    assert len(funcs) == 4
    for name, (lines, meta) in funcs.items():
        assert not _m0_outside_asm(lines), name
        assert meta.get("ScratchSize", 0) == 0, (name, meta)
