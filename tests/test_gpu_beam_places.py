"""TextDecoder.beam_search where there are fewer continuations than beams.

The vocabulary is cut to a few tokens, so that searches of one or two steps have vocab ** count
continuations, each of which has to be there once; the other places hold tokens -1 throughout."""
import itertools

import pytest

torch = pytest.importorskip("torch")

from mold_amd import GgmlDType
from mold_amd.text_decoder import TextDecoder
from tests.test_gpu_text_decoder import CFG, model  # noqa: F401

pytestmark = pytest.mark.gpu
INF = float("inf")
PROMPTS = [[0, 1, 1], [1] * 40, [0]]


def _small(model, vocab):
    """The model with the first `vocab` tokens; its output is the embedding."""
    weights = {k: w for k, w in model[0].items() if k != "output.weight"}
    weights["token_embd.weight"] = weights["token_embd.weight"][:vocab].contiguous()
    return TextDecoder(CFG, weights, pages=300, page_tokens=32, cache_dtype=GgmlDType.BF16)


@pytest.mark.parametrize("vocab,beams,count", [(3, 5, 1), (2, 5, 2), (2, 64, 5), (3, 12, 2), (3, 9, 2)])
def test_places_left_over_have_no_tokens(model, vocab, beams, count):  # noqa: F811
    tokens, scores = _small(model, vocab).beam_search(PROMPTS, beams, count)
    there = vocab ** count
    want = sorted(itertools.product(range(vocab), repeat=count))
    for hypotheses, totals in zip(tokens.tolist(), scores.tolist()):
        assert sorted(tuple(h) for h in hypotheses[:there]) == want
        assert all(h == [-1] * count for h in hypotheses[there:])
        assert all(s > -INF for s in totals[:there]) and all(s == -INF for s in totals[there:])
    # all continuations' probabilities: 1, but for a step's 2^-22 in each logarithm and its rounding, 2^-24 of a total
    # whose mean, the entropy, is at most log 32 = 3.5: below 2^-21 a step
    probability = scores[:, :there].double().exp().sum(1)
    assert (probability - 1).abs().max() <= count * 2.0 ** -20


def test_logits_that_are_no_numbers_end_every_hypothesis(model):  # noqa: F811
    dec = _small(model, 2)
    step, steps = dec.step, []

    def broken(tokens):
        steps.append(tokens)
        logits = step(tokens)
        return logits if len(steps) < 2 else torch.full_like(logits, float("nan"))
    dec.step = broken
    tokens, scores = dec.beam_search(PROMPTS, 2, 3)
    assert (tokens == -1).all() and (scores == -INF).all() and len(steps) == 2


def test_steps_take_tokens_of_the_vocabulary(model):  # noqa: F811
    """Also in the rows of places left over."""
    dec = _small(model, 3)
    step, taken = dec.step, []

    def watched(tokens):
        taken.append(tokens.clone())
        return step(tokens)
    dec.step = watched
    dec.beam_search(PROMPTS, 12, 4)
    assert len(taken) == 3 and all(((t >= 0) & (t < 3)).all() for t in taken)
