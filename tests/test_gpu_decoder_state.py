"""What a text decoder keeps between calls: the buffers that a captured step reads and writes, and
its sequences after a call that failed."""
import pytest

torch = pytest.importorskip("torch")

from mold_amd import GgmlDType
from tests.test_gpu_text_decoder import PROMPTS, VOCAB, _decoder, model  # noqa: F401

pytestmark = pytest.mark.gpu
OTHERS = [[9, 8], list(range(500, 566)), [1, 2, 3, 4, 5, 6, 7, 8, 9], [700] * 4]      # as wide a page table as PROMPTS'


def _capture(dec, token):
    """A step of dec in a graph, and its logits; dec stays where it is."""
    start = dec.lengths.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        dec.step(token)                                      # workspaces of this stream
        dec.lengths.copy_(start)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            logits = dec.step(token)
    torch.cuda.current_stream().wait_stream(s)
    dec.lengths.copy_(start)
    return graph, logits


def _replay_beside(graph, logits, dec, eager, token, count):
    for t in range(count):
        want = eager.step(token)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(logits, want), t
        assert dec.lengths.tolist() == eager.lengths.tolist()
        token.copy_(want.argmax(-1))


def test_captured_step_after_another_prefill(model):
    eager, graphed = _decoder(model, GgmlDType.Q8_0), _decoder(model, GgmlDType.Q8_0)
    token = eager.prefill(PROMPTS, room=20).argmax(-1)
    graphed.prefill(PROMPTS, room=20)
    graph, logits = _capture(graphed, token)
    for prompts in (PROMPTS, OTHERS, PROMPTS[::-1]):
        token.copy_(eager.prefill(prompts, room=20).argmax(-1))
        graphed.prefill(prompts, room=20)
        junk = [torch.full((4, 3), 12345, dtype=torch.int32, device="cuda") for _ in range(8)]
        _replay_beside(graph, logits, graphed, eager, token, 6)
        del junk


def test_captured_step_after_a_prefill_of_another_shape(model):
    """More sequences, or a wider table: the graph of before writes nothing and says so."""
    for prompts, room in ((PROMPTS + [[1, 2]], 20), (PROMPTS, 90)):
        eager, graphed = _decoder(model, GgmlDType.Q8_0), _decoder(model, GgmlDType.Q8_0)
        token = eager.prefill(PROMPTS, room=20).argmax(-1)
        graphed.prefill(PROMPTS, room=20)
        graph, logits = _capture(graphed, token)
        first = eager.prefill(prompts, room=room).argmax(-1)
        graphed.prefill(prompts, room=room)
        held = [c.data.clone() for c in graphed.caches]
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.isnan(logits).all()
        assert all(torch.equal(c.data, h) for c, h in zip(graphed.caches, held))
        again, more = _capture(graphed, first)               # captured anew, it goes on
        _replay_beside(again, more, graphed, eager, first, 4)


def test_a_refused_step_moves_nothing_on(model, monkeypatch):
    """Wrong tokens, and a failure in the middle of a step: the next one gives what it would have."""
    eager, dec = _decoder(model, GgmlDType.BF16), _decoder(model, GgmlDType.BF16)
    token = eager.prefill(PROMPTS, room=20).argmax(-1)
    dec.prefill(PROMPTS, room=20)
    lengths = dec.lengths.tolist()
    for bad in (token[:3], torch.cat([token, token[:1]]), token[:1], token[None], token[:, None], token[0], token.cpu(), token.float(), token > 3):
        with pytest.raises(ValueError):
            dec.step(bad)
        assert dec.lengths.tolist() == lengths
    with monkeypatch.context() as m:
        m.setattr(dec, "_logits", lambda x: 1 / 0)
        with pytest.raises(ZeroDivisionError):
            dec.step(token)
    assert dec.lengths.tolist() == lengths
    for _ in range(3):
        want = eager.step(token)
        assert torch.equal(dec.step(token.int()), want)
        token = want.argmax(-1)


def test_a_failed_prefill_ends_the_sequences_before(model, monkeypatch):
    """Their pages may hold the new prompts' keys by then: a step is refused, a captured one writes
    nothing; the next prefill starts anew.  A prefill that is refused at once changes nothing."""
    eager, dec = _decoder(model, GgmlDType.Q8_0), _decoder(model, GgmlDType.Q8_0)
    token = eager.prefill(PROMPTS, room=20).argmax(-1)
    dec.prefill(PROMPTS, room=20)
    graph, logits = _capture(dec, token)
    for bad in ([], [[1], []], [[1] * 64] * 30):
        with pytest.raises(ValueError):
            dec.prefill(bad)
    _replay_beside(graph, logits, dec, eager, token, 2)
    with monkeypatch.context() as m:
        m.setattr(dec, "_logits", lambda x: 1 / 0)
        with pytest.raises(ZeroDivisionError):
            dec.prefill(OTHERS, room=20)
    with pytest.raises(ValueError):
        dec.step(token)
    held = [c.data.clone() for c in dec.caches]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.isnan(logits).all() and all(torch.equal(c.data, h) for c, h in zip(dec.caches, held))
    token.copy_(eager.prefill(OTHERS, room=20).argmax(-1))
    dec.prefill(OTHERS, room=20)
    _replay_beside(graph, logits, dec, eager, token, 3)


def test_tokens_outside_the_vocabulary_are_refused(model):
    """On the host: on the GPU an index past the embedding is a device assertion, and -1 its last row."""
    dec = _decoder(model, GgmlDType.BF16)
    want = dec.prefill(PROMPTS, room=3)
    for bad in (VOCAB, -1, 1 << 40):
        with pytest.raises(ValueError):
            dec.prefill([[1, 2], [3, bad, 4]])
    assert dec.lengths.tolist() == [len(p) for p in PROMPTS]
    assert torch.equal(dec.prefill(PROMPTS, room=3), want)
    dec.prefill([[0, VOCAB - 1]])


def test_no_tokens_and_negative_counts(model):
    dec = _decoder(model, GgmlDType.BF16)
    for count in (0, 1, 2):
        assert dec.generate(PROMPTS, count).shape == (len(PROMPTS), count)
    for call in (lambda: dec.generate(PROMPTS, -1), lambda: dec.prefill(PROMPTS, room=-1), lambda: dec.prefill([[1] * 33], room=-2)):
        with pytest.raises(ValueError):
            call()
