"""TextDecoder.beam_search: the operators of a step run together, as a search uses them.

A hypothesis' log probability has to be the sum over its tokens that the decoder gives when the
same tokens are stepped without any reordering, in rows of their own.  Both sides read the same
weights and caches of the same values; what may differ is the order of sums in attention, a bf16
rounding (2^-8) here and there of what goes into a layer's linears, far below the 2e-2 by which a step's
logits are allowed to be off a float64 model (test_gpu_text_decoder), so 2e-2 of the logits' size a
step is asserted.  A row with another row's cache is off by their whole size."""
from dataclasses import replace

import pytest

torch = pytest.importorskip("torch")

from mold_amd import GgmlDType
from mold_amd.text_decoder import TextDecoder
from tests.test_gpu_text_decoder import CFG, PROMPTS, VOCAB, _decoder, model  # noqa: F401

pytestmark = pytest.mark.gpu


def _forced(dec, prompts, hypotheses):
    """float64 [n * beams, count] log probabilities of given tokens, and the logits' size."""
    n, beams, count = hypotheses.shape
    rows = [p for p in prompts for _ in range(beams)]
    logits, out, size = dec.prefill(rows, room=count), [], 0.0
    for t in range(count):
        token = hypotheses[:, :, t].reshape(-1)
        out.append(torch.gather(torch.log_softmax(logits.double(), -1), 1, token[:, None])[:, 0])
        size = max(size, logits.double().square().mean().sqrt().item())
        logits = dec.step(token)
    return torch.stack(out, 1), size


@pytest.mark.parametrize("dtype", [GgmlDType.BF16, GgmlDType.Q8_0, GgmlDType.Q4_0], ids=lambda t: t.name)
@pytest.mark.parametrize("beams", [2, 5])
def test_hypotheses_have_their_probability(model, dtype, beams):  # noqa: F811
    """Past the end of a page of 32, from prompts that fill none, a part or two of them."""
    prompts, count = PROMPTS + [list(range(64))], 37
    dec = _decoder(model, dtype, pages=200)
    tokens, scores = dec.beam_search(prompts, beams, count)
    assert tokens.shape == (len(prompts), beams, count) and scores.shape == (len(prompts), beams)
    assert (scores[:, 1:] <= scores[:, :-1]).all() and torch.isfinite(scores).all()
    for hypotheses in tokens.tolist():
        assert len({tuple(h) for h in hypotheses}) == beams
    each, size = _forced(_decoder(model, dtype, pages=400), prompts, tokens)
    off = (each.sum(1).view_as(scores) - scores.double()).abs()
    assert off.max() <= count * 2e-2 * size, (off.max(), size)
    assert dec.lengths.tolist() == [len(p) + count - 1 for p in prompts for _ in range(beams)]


def test_one_beam_is_the_greedy_choice(model):  # noqa: F811
    dec = _decoder(model, GgmlDType.BF16, pages=40)
    want = dec.generate(PROMPTS, 12)
    tokens, scores = dec.beam_search(PROMPTS, 1, 12)
    assert torch.equal(tokens[:, 0], want) and (scores < 0).all()


def test_the_first_step_finds_the_most_probable(model):  # noqa: F811
    dec = _decoder(model, GgmlDType.BF16, pages=60)
    logits = dec.prefill(PROMPTS)
    want = torch.log_softmax(logits.double(), -1).topk(4)
    tokens, scores = dec.beam_search(PROMPTS, 4, 1)
    assert torch.equal(tokens[:, :, 0], want.indices)
    torch.testing.assert_close(scores.double(), want.values, rtol=2.0 ** -23, atol=2.0 ** -22)


def test_stopped_hypotheses_repeat_their_stop(model):  # noqa: F811
    dec = _decoder(model, GgmlDType.BF16, pages=60)
    free, _ = dec.beam_search(PROMPTS, 3, 8)
    stop = int(free[0, 0, 2])
    tokens, scores = dec.beam_search(PROMPTS, 3, 8, stop=stop)
    ended = (tokens == stop).cumsum(-1) > 0
    assert ended.any() and (tokens[ended] == stop).all()
    each, size = _forced(_decoder(model, GgmlDType.BF16, pages=400), PROMPTS, tokens)
    after = torch.cat([torch.zeros_like(ended[..., :1]), ended[..., :-1]], -1).view_as(each)
    off = (torch.where(after, 0.0, each).sum(1).view_as(scores) - scores.double()).abs()
    assert off.max() <= 8 * 2e-2 * size


def test_edges(model):  # noqa: F811
    dec = _decoder(model, GgmlDType.BF16, pages=60)
    tokens, scores = dec.beam_search(PROMPTS, 3, 0)
    assert tokens.shape == (4, 3, 0) and (scores == 0).all()
    for call in (lambda: dec.beam_search(PROMPTS, 0, 4), lambda: dec.beam_search(PROMPTS, 65, 4), lambda: dec.beam_search(PROMPTS, 2, -1), lambda: dec.beam_search([], 2, 3),
                 lambda: dec.beam_search(PROMPTS, 30, 40), lambda: dec.beam_search([[VOCAB]], 2, 2), lambda: dec.beam_search(PROMPTS, 2, 3, stop=VOCAB), lambda: dec.beam_search(PROMPTS, 2, 1, stop=-1)):
        with pytest.raises(ValueError):
            call()
    again = dec.beam_search(PROMPTS, 3, 5)
    assert all(torch.equal(a, b) for a, b in zip(again, dec.beam_search(PROMPTS, 3, 5)))


def test_a_search_step_in_a_graph(model):  # noqa: F811
    """Selection, reordering and the next step, replayed, go on as the eager search does."""
    from mold_amd.beams import select_beams
    beams, n = 3, len(PROMPTS)

    def start(dec):
        logits = dec.prefill(PROMPTS, room=40, beams=beams)
        scores, _, tokens = select_beams(logits[:, None], torch.zeros((n, 1), device="cuda"), beams)
        return dec.step(tokens.reshape(-1)), scores

    def go_on(dec, logits, scores):
        scores, parents, tokens = select_beams(logits.view(n, beams, -1), scores)
        dec._states.reorder(dec.table, dec.lengths, parents)
        return dec.step(tokens.reshape(-1)), scores, tokens
    eager, graphed = _decoder(model, GgmlDType.Q8_0, pages=80), _decoder(model, GgmlDType.Q8_0, pages=80)
    want = start(eager)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        logits, scores = start(graphed)
        go_on(graphed, logits, scores)                       # workspaces of this stream
        logits, scores = start(graphed)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = go_on(graphed, logits, scores)
            logits.copy_(out[0])
            scores.copy_(out[1])
    torch.cuda.current_stream().wait_stream(s)
    for _ in range(30):
        want = go_on(eager, *want[:2])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_head_norms_in_bf16(model):  # noqa: F811
    """Weights that come in another type than the documented float32 are taken by their values."""
    weights = {k: w.bfloat16() if k.endswith(("_q_norm.weight", "_k_norm.weight")) else w for k, w in model[0].items()}
    same = {k: w.float() if k.endswith(("_q_norm.weight", "_k_norm.weight")) else w for k, w in weights.items()}
    a, b = (_decoder((w, None), GgmlDType.BF16) for w in (weights, same))
    assert torch.equal(a.prefill(PROMPTS, room=1), b.prefill(PROMPTS, room=1))
    token = torch.arange(len(PROMPTS), device="cuda")
    assert torch.equal(a.step(token), b.step(token))


def test_more_layers_than_are_reordered_at_once(model):  # noqa: F811
    """A decoder of 257 layers runs; beams of it are refused before anything ends."""
    layers = 257
    weights = {k: w for k, w in model[0].items() if not k.startswith("blk.")}
    for i in range(layers):
        weights.update({k.replace("blk.0.", f"blk.{i}."): w for k, w in model[0].items() if k.startswith("blk.0.")})
    dec = TextDecoder(replace(CFG, layers=layers), weights, pages=8, page_tokens=32, cache_dtype=GgmlDType.BF16)
    assert dec.prefill(PROMPTS[:2], room=4).shape == (2, VOCAB)
    with pytest.raises(ValueError):
        dec.beam_search(PROMPTS[:1], 2, 3)
    assert torch.isfinite(dec.step(torch.tensor([1, 2], device="cuda"))).all()
