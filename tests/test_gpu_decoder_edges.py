"""TextDecoder at the ends of its configuration."""
from dataclasses import replace

import pytest

torch = pytest.importorskip("torch")

from mold_amd import GgmlDType
from mold_amd.text_decoder import TextDecoder, rms_norm
from tests.test_gpu_text_decoder import CFG, PROMPTS, VOCAB, model  # noqa: F401

pytestmark = pytest.mark.gpu


def test_no_layers(model):  # noqa: F811
    """The embedding, the last norm and the output, each token by itself.  In float32: sums of 512 products, 2^-15 of
    the products' sizes, which are 16 times the result's size, so below 2^-10 of that with what goes into them."""
    weights = {k: w for k, w in model[0].items() if not k.startswith("blk.") and k != "output.weight"}
    dec = TextDecoder(replace(CFG, layers=0), weights, pages=10, page_tokens=32, cache_dtype=GgmlDType.BF16)
    embedding = weights["token_embd.weight"].double()

    def want(tokens):
        return rms_norm(embedding[tokens], weights["output_norm.weight"].double(), CFG.eps).double() @ embedding.t()

    def same(got, tokens):
        w = want(tokens)
        assert got.shape == (len(PROMPTS), VOCAB) and (got.double() - w).abs().max() <= 2.0 ** -10 * w.square().mean().sqrt()
    last = torch.tensor([p[-1] for p in PROMPTS], device="cuda")
    same(dec.prefill(PROMPTS, room=3), last)
    step = torch.tensor([1, 2, 3, 4], device="cuda")
    same(dec.step(step), step)
    assert dec.lengths.tolist() == [len(p) + 1 for p in PROMPTS]
    assert dec.generate(PROMPTS, 1)[:, 0].tolist() == want(last).argmax(-1).tolist()
