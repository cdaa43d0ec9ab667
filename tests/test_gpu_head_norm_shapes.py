"""Head norms whose weights are not one vector of a head's size: one of each head, or a number for
all values.  They broadcast over [heads, head_dim], as the float64 model of test_gpu_text_decoder does it;
bounds as there."""
import pytest

torch = pytest.importorskip("torch")

from mold_amd import GgmlDType
from mold_amd.text_decoder import TextDecoder
from tests.test_gpu_text_decoder import CFG, PROMPTS, _err, _reference, model  # noqa: F401

pytestmark = pytest.mark.gpu
SHAPES = {"q": {"q": (CFG.heads, CFG.head_dim)}, "k": {"k": (CFG.kv_heads, CFG.head_dim)}, "number": {"q": (), "k": (1,)},
          "head": {"q": (CFG.heads, 1), "k": (1, CFG.head_dim)}}


@pytest.mark.parametrize("kind", SHAPES)
@pytest.mark.parametrize("dtype,bound", [(GgmlDType.BF16, 2e-2), (GgmlDType.Q8_0, 5e-2)], ids=lambda x: getattr(x, "name", ""))
def test_against_float64(model, kind, dtype, bound):  # noqa: F811
    weights, dense = dict(model[0]), dict(model[1])
    g = torch.Generator(device="cuda").manual_seed(5)
    for i in range(CFG.layers):
        for which, shape in SHAPES[kind].items():
            name = f"blk.{i}.attn_{which}_norm.weight"
            weights[name] = 1 + 0.3 * torch.randn(shape, device="cuda", generator=g)
            dense[name] = weights[name].double()
    dec = TextDecoder(CFG, weights, pages=40, page_tokens=32, cache_dtype=dtype)
    logits = dec.prefill(PROMPTS, room=4)
    more = [[7, 9, 400, 2], [1, 2, 3, 4], [999, 0, 5, 6], [8, 8, 8, 8]]
    refs = [_reference(dense, p + m) for p, m in zip(PROMPTS, more)]
    for i, p in enumerate(PROMPTS):
        assert _err(logits[i], refs[i][len(p) - 1]) < 2e-2, i
    for t in range(4):
        logits = dec.step(torch.tensor([m[t] for m in more], device="cuda"))
        for i, p in enumerate(PROMPTS):
            assert _err(logits[i], refs[i][len(p) + t]) < bound, (t, i)
