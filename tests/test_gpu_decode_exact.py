"""mq_cache_attention loses nothing before its output's rounding: keys, values and probabilities
enter the products to 2^-16 and better, so that every element is the float64 result over what the
cache holds, rounded to bf16 once, up to what float32 sums leave.

The bound, element by element, with A = sum_t p_t |v_t| of the row: half a unit of the bf16
result's last place (2^(e - 8) for a result in 2^e .. 2^(e + 1)), and 2^-14 A for
  the probabilities' second bf16 part        2^-16 (2^-7 left by the first, 2^-9 of that by the second)
  their exponents, |scale q . k| up to 16    16 x 2^-23 x 3 (product, sums, log2(e)) < 2^-17.4
  float32 sums of up to 300 tokens           2^-24 x 2 x 10 tiles, and the joins
With the second part lost the error is 2^-9 A on average and past half a unit in many elements.

Q4_0's operands are n + 128 and -136 for a stored n = 0 .. 15, whose products cancel in float32:
there the terms summed are up to 143 C and not A, with C = sum_t p_t |d_t| of the value blocks'
scales.  Each of a tile's four products rounds sums of that size, once for each of the four groups
of eight tokens in it: 16 x 143 x 2^-24 C beside the bound above, 2^-12.8 C, where A is 4 C or
more for most elements."""
import pytest

torch = pytest.importorskip("torch")

from mold_amd import GgmlDType
from tests.test_gpu_decode_attention import _Batch


def _over(out, p, v, t):
    """How far `out` [heads, dim] is past the bound at worst; p [heads, tokens] and v [heads, tokens, dim] in float64."""
    exact, size = (p.unsqueeze(1) @ v).squeeze(1), (p.unsqueeze(1) @ v.abs()).squeeze(1)
    half = torch.exp2(torch.floor(torch.log2(exact.abs().clamp(min=1e-30))) - 8)
    over = (out - exact).abs() - half - 2.0 ** -14 * size
    if t == GgmlDType.Q4_0:                                  # d: a block's largest magnitude is 8 |d|
        d = v.unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True).expand(-1, -1, -1, 32).flatten(-2) / 8
        over -= 16 * 143 * 2.0 ** -24 * (p.unsqueeze(1) @ d).squeeze(1)
    return over.max().item()


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("t", [GgmlDType.BF16, GgmlDType.Q8_0, GgmlDType.Q4_0], ids=lambda t: t.name)
@pytest.mark.parametrize("room", [0, 4000])
def test_rounded_once(t, dim, room):
    """In the form for short page tables and (with `room`) the one for long ones."""
    lengths = [1, 2, 3, 5, 17, 32, 33, 64, 90, 300]
    b = _Batch(lengths, 8, 2, dim, t)
    b.table = torch.nn.functional.pad(b.table, (0, room // b.page), value=-1)
    out = b.run().double().cpu()
    for i, slots in enumerate(b.slots):
        k, v = (x.double().cpu().repeat_interleave(4, 1).transpose(0, 1).contiguous() for x in b.cache.read(slots, torch.float32))
        s = (k @ b.q[i].double().cpu().unsqueeze(2)).squeeze(2) * dim ** -0.5
        assert s.abs().max() < 16
        over = _over(out[i], torch.softmax(s, -1), v, t)
        assert over <= 0, (lengths[i], over)


@pytest.mark.parametrize("t", [GgmlDType.BF16, GgmlDType.Q8_0, GgmlDType.Q4_0], ids=lambda t: t.name)
@pytest.mark.parametrize("n", [3, 33, 300])
def test_the_bound_tells_one_rounding_from_two(t, n):
    """Probabilities (of the block types, times their block's scale) rounded to bf16 once, without
    their second part, on the CPU: far past the bound; in float32: within it."""
    g = torch.Generator().manual_seed(n)
    p = torch.softmax(torch.randn((8, n), generator=g, dtype=torch.float64), -1)
    v = torch.randn((8, n, 64), generator=g)
    if t == GgmlDType.BF16:
        v = v.bfloat16().double()
        weights, values = p.unsqueeze(2), v
    else:
        top = 127 if t == GgmlDType.Q8_0 else 8
        d = (v.unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True) / top).half().double().expand(-1, -1, -1, 32).flatten(-2)
        values = (v / d).round().clamp(-top, top)
        v, weights = values * d, p.unsqueeze(2) * d
    once = lambda dtype: (weights.to(dtype).double() * values).sum(1).bfloat16().double()
    assert _over(once(torch.float32), p, v, t) <= 0 < _over(once(torch.bfloat16), p, v, t)
