"""Beam search over a decoder's logits and paged caches, run by libmoldq (mq_beam_select and
mq_beam_reorder in include/moldq.h).

A search of `beams` hypotheses of each request keeps them as rows request * beams + beam of the
page table: after each step select_beams picks the continuations, BeamStates.reorder
makes each row's cache its parent's, and the picked tokens are the next step's.  Totals are
plain sums of log probabilities; a beam that has given its stop token keeps its total.

Everything runs on torch's current stream of the tensors' device, reads lengths and parents
there, and may be captured in a graph.  There is no counterpart in the reference, which samples
one sequence (crates/mold-inference/src/expand.rs:200-203).
"""
from __future__ import annotations

from typing import Sequence

import torch

from . import _lib
from .fused import recorded
from .quantized import _dtype_code
from .text_attention import KvCache, _run_on

_MAX_STRIDE = 1 << 40


def select_beams(logits, scores, count=None, last=None, stop=None):
    """The `count` (default: as many as beams) best continuations of each request: logits [n, beams,
    vocab] (bf16 or f32) after its beams, scores f32 [n, beams] their totals so far -> (totals f32,
    parents int32, tokens int64), each [n, count], the largest scores[beam] +
    log_softmax(logits[beam])[token] first; ties go to the lower beam, within a beam to the lower token
    (totals of different beams within some 2^-22 of each other may come in either order). With `stop`, a
    beam whose `last` token (int64 [n, beams]) was `stop` has that one continuation, at its total as it
    is. A beam of a score that is not finite or with a NaN or plus infinity among its logits has none;
    places left over have total -inf, parent 0, token -1. Up to 2^20 requests, fewer than 2^24 rows of
    logits."""
    if recorded(logits, scores):
        raise ValueError("select_beams: inference only, nothing may record the call")
    if logits.dim() != 3 or logits.dtype not in (torch.float32, torch.bfloat16) or logits.device.type != "cuda":
        raise ValueError("select_beams: logits must be bf16 or f32 [requests, beams, vocab] on a GPU")
    n, beams, vocab = logits.shape
    device, count = logits.device, beams if count is None else int(count)
    if not 1 <= beams <= _lib.MQ_MAX_BEAMS or not 1 <= count <= _lib.MQ_MAX_BEAMS or vocab < 1:
        raise ValueError(f"select_beams: 1 to {_lib.MQ_MAX_BEAMS} beams and continuations, of at least one token; got {beams}, {count}, {vocab}")
    if n > 1 << 20 or n * beams >= 1 << 24:
        raise ValueError(f"select_beams: up to 2^20 requests, fewer than 2^24 rows of logits; got {n} of {beams} beams")
    if (last is None) != (stop is None):
        raise ValueError("select_beams: last and stop go together")
    if stop is not None and not 0 <= stop < vocab:
        raise ValueError(f"select_beams: stop {stop} is not one of {vocab} tokens")
    if scores.dtype is not torch.float32 or scores.shape != (n, beams) or scores.device != device:
        raise ValueError(f"select_beams: scores must be float32 [{n}, {beams}] on {device}")
    if not scores.is_contiguous():
        scores = scores.contiguous()
    last_at = None
    if last is not None:
        if last.dtype is not torch.int64 or last.shape != (n, beams) or last.device != device:
            raise ValueError(f"select_beams: last must be int64 [{n}, {beams}] on {device}")
        if not last.is_contiguous():
            last = last.contiguous()
        last_at = last.data_ptr()
    sn, sb, sv = logits.stride()
    if sv != 1 and vocab > 1 or sn >= _MAX_STRIDE or sb >= _MAX_STRIDE:
        logits = logits.contiguous()
        sn, sb, _ = logits.stride()
    if count == beams:
        totals = torch.empty_like(scores)
        parents, tokens = torch.empty_like(scores, dtype=torch.int32), torch.empty_like(scores, dtype=torch.int64)
    else:
        totals = scores.new_empty((n, count))
        parents, tokens = scores.new_empty((n, count), dtype=torch.int32), scores.new_empty((n, count), dtype=torch.int64)
    if n:
        lib, code = _lib.load(), _dtype_code(logits.dtype)
        nbytes = lib.mq_beam_select_scratch_size(n, beams, vocab, count, code)
        scratch = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None     # freed to this stream
        _run_on(device, lib.mq_beam_select, logits.data_ptr(), code, n, beams, vocab, sn, sb, scores.data_ptr(),
                last_at, 0 if stop is None else stop, count, totals.data_ptr(), parents.data_ptr(),
                tokens.data_ptr(), scratch.data_ptr() if nbytes else None, nbytes)
    return totals, parents, tokens


class BeamStates:
    """The caches of a model's layers (alike, each its own memory), whose sequences are reordered together."""

    def __init__(self, caches: Sequence[KvCache]):
        self.caches = list(caches)
        if not 1 <= len(self.caches) <= 256:
            raise ValueError(f"BeamStates: 1 to 256 caches, got {len(self.caches)}")
        first = self.caches[0]
        like = lambda c: (c.device, c.dtype, c.pages, c.kv_heads, c.head_dim, c.page_tokens)
        if any(like(c) != like(first) for c in self.caches):
            raise ValueError("BeamStates: the caches of a model's layers are alike")
        if first.pages and len({c.data.data_ptr() for c in self.caches}) < len(self.caches):
            raise ValueError("BeamStates: a cache is there twice")
        self.device = first.device
        self.c = (_lib.KvCacheC * len(self.caches))(*(c.c for c in self.caches))
        self._streams = set()      # that all caches know to use them

    def reorder(self, page_table, lengths, parents):
        """Beam j of each of up to 2^20 requests goes on from beam parents[n, j] (int32 [n, beams]; itself if it
        is no beam): its row of page_table (int32 [n * beams, pages], changed in place) and the tokens so
        far, lengths (int32 [n * beams], the same for a request's beams), become the parent's.
        Whole pages are shared; of the last, partial one, which no two rows may share before,
        each row has its own after it too, copied where a parent has several children."""
        if recorded(page_table, lengths, parents):
            raise ValueError("BeamStates.reorder: inference only, nothing may record the call")
        device = self.device
        if parents.dtype is not torch.int32 or parents.dim() != 2 or parents.device != device or not 1 <= parents.shape[1] <= _lib.MQ_MAX_BEAMS:
            raise ValueError(f"BeamStates.reorder: parents must be int32 [requests, beams] on {device}, of 1 to {_lib.MQ_MAX_BEAMS} beams")
        n, beams = parents.shape
        if page_table.dtype is not torch.int32 or page_table.dim() != 2 or page_table.shape[0] != n * beams or page_table.device != device:
            raise ValueError(f"BeamStates.reorder: page_table must be int32 [{n * beams}, pages] on {device}")
        if lengths.dtype is not torch.int32 or lengths.shape != (n * beams,) or lengths.device != device:
            raise ValueError(f"BeamStates.reorder: lengths must be int32 [{n * beams}] on {device}")
        width = page_table.shape[1]
        if n * beams > 1 and (page_table.stride(0) < width or width > 1 and page_table.stride(1) != 1):
            raise ValueError("BeamStates.reorder: page_table's rows must be apart, each one run of memory: they are changed in place")
        parents = parents if parents.is_contiguous() else parents.contiguous()
        lengths = lengths if lengths.is_contiguous() else lengths.contiguous()
        if n == 0 or beams == 1:
            return
        lib = _lib.load()
        nbytes = lib.mq_beam_reorder_scratch_size(n, beams)
        scratch = torch.empty(nbytes, dtype=torch.uint8, device=device)     # freed to this stream
        stream = torch._C._cuda_getCurrentRawStream(device.index)
        if stream not in self._streams:
            for c in self.caches:
                c._on.seen(stream)
            self._streams.add(stream)
        _run_on(device, lib.mq_beam_reorder, self.c, len(self.caches), page_table.data_ptr(), page_table.stride(0), width,
                lengths.data_ptr(), parents.data_ptr(), n, beams, scratch.data_ptr(), nbytes)
        if not page_table.is_inference():      # which has no version
            torch.autograd.graph.increment_version(page_table)      # written in place, as a copy_ tells autograd
