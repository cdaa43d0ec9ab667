"""mq_beam_select at the most requests and rows that it documents, and past them."""
import math

import pytest

torch = pytest.importorskip("torch")

from mold_amd import _lib
from mold_amd.beams import select_beams


@pytest.mark.gpu
@pytest.mark.parametrize("n,beams,vocab", [((1 << 18) - 1, 64, 5), (1 << 20, 15, 3), (1 << 20, 8, 2), (1 << 20, 1, 2)])
def test_as_many_rows_as_are_documented(n, beams, vocab):
    """One logit of 4 beside others of 0: each request's best is the one beam whose score is not lower."""
    g = torch.Generator(device="cuda").manual_seed(n + beams)
    best = torch.randint(0, beams, (n,), device="cuda", generator=g)
    scores = torch.full((n, beams), -9.0, device="cuda")
    scores.scatter_(1, best[:, None], 0.0)
    token = torch.randint(0, vocab, (n, 1, 1), device="cuda", generator=g)
    logits = (torch.arange(vocab, device="cuda") == token).to(torch.bfloat16).mul_(4).expand(n, beams, vocab)
    totals, parents, tokens = select_beams(logits, scores, 1)
    assert torch.equal(parents[:, 0].long(), best) and torch.equal(tokens[:, 0], token[:, 0, 0])
    want = -math.log1p((vocab - 1) * math.exp(-4))      # within the bound of test_gpu_beams
    assert (totals.double() - want).abs().max() <= 2.0 ** -22 + 2.0 ** -23 * abs(want)


@pytest.mark.gpu
@pytest.mark.parametrize("n,beams", [((1 << 20) + 1, 1), (1 << 18, 64), (1 << 20, 16)])
def test_more_are_refused(n, beams):
    logits, scores = torch.zeros((1, 1, 4), device="cuda").expand(n, beams, 4), torch.zeros((1, 1), device="cuda").expand(n, beams)
    with pytest.raises(ValueError, match="2\\^24"):
        select_beams(logits, scores, 1)


def test_the_library_refuses_them():
    """On the CPU: before anything is launched; what is refused needs no scratch."""
    lib, a = _lib.load(), 4096
    args = dict(logits=a, dtype=0, requests=1 << 18, beams=64, vocab=100, request_stride=6400, beam_stride=100, scores=a, last=None, stop=0, count=2,
                out_scores=a, parents=a, tokens=a, scratch=a, scratch_bytes=1 << 40, stream=None)
    for n, beams in (((1 << 20) + 1, 1), (1 << 18, 64), (1 << 20, 16)):
        assert lib.mq_beam_select(*{**args, "requests": n, "beams": beams}.values()) == _lib.MQ_E_INVALID, (n, beams)
        assert lib.mq_beam_select_scratch_size(n, beams, 100, 64, 0) == 0, (n, beams)
    assert lib.mq_beam_select_scratch_size((1 << 18) - 1, 64, 100, 64, 0) == ((1 << 18) - 1) * 64 * (16 + 8 * 64)      # a run and its keys, past 32 bits
