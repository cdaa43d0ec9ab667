"""TextDecoder at the ends of its configuration."""
from dataclasses import replace

import pytest

torch = pytest.importorskip("torch")

from mold_amd import Device, GgmlDType, QTensor, text_decoder
from mold_amd.text_decoder import TextConfig, TextDecoder, rms_norm
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


def _same_start(a, b):
    """The sequences' places, and what every call gives, of two decoders."""
    prompts = [[i % 7, 3, i % 5][:1 + i % 3] * (1 + 40 * (i % 11 == 0)) for i in range(50)]
    assert torch.equal(a.prefill(prompts, room=40), b.prefill(prompts, room=40))
    assert torch.equal(a.table, b.table) and torch.equal(a.lengths, b.lengths)
    for i in range(3):
        token = (torch.arange(50, device="cuda") + i) % VOCAB
        assert torch.equal(a.step(token), b.step(token)) and torch.equal(a.lengths, b.lengths)


@pytest.mark.parametrize("most", [1, 7, 16, 49])
def test_places_in_several_calls(model, most, monkeypatch):  # noqa: F811
    """Sequences placed a few at a time lie where those placed at once do."""
    a, b = (TextDecoder(CFG, model[0], pages=300, page_tokens=32, cache_dtype=GgmlDType.Q8_0) for _ in range(2))
    place, extend = b._place, b._extend

    def few(call):
        def run(*args):
            with monkeypatch.context() as m:
                m.setattr(text_decoder, "_MOST", most)
                return call(*args)
        return run
    b._place, b._extend = few(place), few(extend)
    _same_start(a, b)


def test_more_sequences_than_one_call_places():
    """2^20 and a few, as before tables were made on the GPU: rows of the same prompt alike."""
    hidden, vocab, n = 256, 64, (1 << 20) + 5
    g = torch.Generator(device="cuda").manual_seed(0)
    rand = lambda *s: torch.randn(s, device="cuda", generator=g) * 0.05
    weights = {"token_embd.weight": rand(vocab, hidden) * 20, "output_norm.weight": 1 + rand(hidden), "blk.0.attn_norm.weight": 1 + rand(hidden),
               "blk.0.ffn_norm.weight": 1 + rand(hidden)}
    for name, rows, columns in (("attn_q", 128, hidden), ("attn_k", 64, hidden), ("attn_v", 64, hidden), ("attn_output", hidden, 128), ("ffn_gate", 256, hidden),
                                ("ffn_up", 256, hidden), ("ffn_down", hidden, 256)):
        weights[f"blk.0.{name}.weight"] = QTensor.quantize(Device(0), rand(rows, columns), GgmlDType.Q8_0)
    config = TextConfig(hidden, 2, 1, 64, 1)
    small, dec = (TextDecoder(config, weights, pages=pages, page_tokens=32, cache_dtype=GgmlDType.Q4_0) for pages in (vocab, n))
    want, got = small.prefill([[i] for i in range(vocab)], room=2), dec.prefill([[i % vocab] for i in range(n)], room=2)
    which = torch.arange(n, device="cuda") % vocab
    for _ in range(2):
        # one token's activations in linears of other row counts: their roundings to bf16, as in test_gpu_text_decoder
        assert ((got - want[which]).norm(dim=1) <= 2e-2 * want[which].norm(dim=1)).all()
        assert torch.equal(dec.table[:, 0], torch.arange(n, device="cuda", dtype=torch.int32))
        want, got = small.step(torch.arange(vocab, device="cuda")), dec.step(which)
    assert (dec.lengths == 3).all()
    with pytest.raises(ValueError, match="2\\^20"):
        dec.prefill([[1]] * n, beams=2)
