"""A GGUF text decoder on the library's linears and text attention: prompts in, tokens out.

What mold's prompt expansion runs through candle's quantized_qwen3::ModelWeights
(crates/mold-inference/src/expand.rs:200-203): RmsNorm, grouped-head attention with rotary
halves and optional q/k head norms, and a SwiGLU MLP, with tensor names as GGUF files give
them (TextConfig.from_metadata and gguf.Content.var_builder make one of a file).  `prefill`
takes a batch of prompts packed without padding, `step` one new token of each sequence; both
write their keys and values into one paged cache (quantized where its type is a block type)
that `step` attends over.  Projections are QMatMul; the norms and rotation of q and k, their way
into the cache, pages and slots, and attention are text_attention; the other norms and the activation are
torch operations in float32.  `generate` takes the likeliest token each time, `beam_search` keeps
several hypotheses of each prompt (beams), whose cached prompts share their whole pages.

`step` makes no host synchronization: lengths and page table stay on the device, so it can be
captured in a graph.  The graph goes on to a later prefill's sequences if there are as many and
their page table is as wide; otherwise its replays write nothing and give NaN, and a step has to
be captured anew.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, Optional, Sequence

import torch

from ._lib import MQ_MAX_BEAMS
from .beams import BeamStates, select_beams
from .quantized import GgmlDType, QMatMul, QTensor
from .text_attention import KvCache, Placed, PromptPlan, prompt_attention

_MOST = 1 << 20      # sequences that place and extend take at once

@dataclass(frozen=True)
class TextConfig:
    hidden: int
    heads: int
    kv_heads: int
    head_dim: int
    layers: int
    rope_theta: float = 1e6
    eps: float = 1e-6

    @classmethod
    def from_metadata(cls, metadata: Dict[str, object]) -> "TextConfig":
        """A GGUF file's (Content.metadata), by the keys of its architecture."""
        arch = metadata["general.architecture"]
        get = lambda key, default=None: metadata.get(f"{arch}.{key}", default)
        sizes = {key: get(key) for key in ("embedding_length", "attention.head_count", "block_count")}
        if None in sizes.values():
            raise ValueError(f"TextConfig: the metadata has no {', '.join(f'{arch}.{k}' for k, v in sizes.items() if v is None)}")
        hidden, heads, layers = sizes.values()
        return cls(hidden, heads, get("attention.head_count_kv", heads), get("attention.key_length", hidden // heads), layers,
                   get("rope.freq_base", cls.rope_theta), get("attention.layer_norm_rms_epsilon", cls.eps))


def rms_norm(x, weight, eps: float):
    """float32 RmsNorm over the last axis."""
    x = x.float()
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weight


def rotate(x, cos, sin):
    """Rotary embedding of the halves of each head: x [tokens, heads, dim], cos and sin [tokens, dim / 2] -> float32.
    The plain form, for angles that a caller has; the decoder's own are taken by KvCache.append_rotated."""
    a, b = x.float().chunk(2, -1)
    c, s = cos[:, None], sin[:, None]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


class TextDecoder:
    """weights: {GGUF name: QTensor (as Content.var_builder gives them all) or float32 tensor};
    `output.weight` falls back to the embedding, `attn_{q,k}_norm` and biases are optional.
    Projections of a block type stay as they are; the embedding, norms, biases and whatever is
    stored dense are held in float32.  One layer's cache each, `pages` pages of `page_tokens` tokens."""

    def __init__(self, config: TextConfig, weights: Dict[str, object], pages: int, page_tokens: int = 64,
                 cache_dtype: GgmlDType = GgmlDType.Q8_0, device="cuda"):
        self.config = config
        self.weights = {name: self._dense(name, w) if isinstance(w, QTensor) else w for name, w in weights.items()}
        if self._blocks(weights["token_embd.weight"]):
            self.weights.setdefault("output.weight", weights["token_embd.weight"])
        self.device = torch.device(device)
        self.page_tokens, self.pages = page_tokens, pages
        self.caches = [KvCache(pages, config.kv_heads, config.head_dim, page_tokens, cache_dtype, device)
                       for _ in range(config.layers)]
        # where tokens go is the same in every layer's, and without layers all the same
        self._placing = self.caches[0] if self.caches else KvCache(pages, config.kv_heads, config.head_dim, page_tokens, cache_dtype, device)
        self.table = self.lengths = self._buffers = None
        self._captured, self._retired = False, []     # what graphs of earlier batches hold
        half = config.head_dim // 2
        self._states = None       # of the caches, once beams are reordered
        self._inv_freq = config.rope_theta ** (-torch.arange(half, device=device, dtype=torch.float32) / half)

    @staticmethod
    def _blocks(w) -> bool:
        return isinstance(w, QTensor) and w.dtype().is_quantized

    def _dense(self, name: str, w: QTensor):
        """w as it is used: a projection in blocks as it is, anything else in float32, a vector as one."""
        if name.endswith("norm.weight") or name.endswith(".bias"):
            return w.dequantize().reshape(-1)
        return w if self._blocks(w) and name != "token_embd.weight" else w.dequantize()

    def _linear(self, name: str, x, out_dtype=torch.float32):
        bias = self.weights.get(name + ".bias")
        w = self.weights[name + ".weight"]
        if isinstance(w, QTensor):
            return QMatMul(w).forward(x, bias=bias, out_dtype=out_dtype)
        y = x.float() @ w.t()
        return (y if bias is None else y + bias).to(out_dtype)

    def _head_norm(self, name: str, x):
        """x and the weight of the norm that goes with its rotation, f32 [head_dim]; a weight that varies over
        the heads, or is one for the whole head, is applied to x here, which gives float32."""
        weight = self.weights.get(name)
        if weight is None or weight.shape[-1:].numel() == weight.numel() == self.config.head_dim:
            return x, weight if weight is None else weight.reshape(-1).float()
        return rms_norm(x, weight, self.config.eps).float(), None

    def _beam_states(self):
        if self._states is None:
            self._states = BeamStates(self.caches)
        return self._states

    def _place(self, lengths, need, per, room, beams):
        """Where prompts of these lengths go, which need so many pages each of the cache's."""
        parts, page, row = [], 0, 0
        for i in range(0, len(lengths), _MOST):
            some, pages = lengths[i:i + _MOST], sum(need[i:i + _MOST])
            order = torch.arange(page, page + pages, dtype=torch.int32, device=self.device) if page else None
            at = self._placing.place(torch.tensor(some, dtype=torch.int32).to(self.device), sum(some), per, room, beams, order)
            parts.append(at._replace(last=at.last + row) if row else at)
            page, row = page + pages, row + sum(some)
        return parts[0] if len(parts) == 1 else Placed(*(torch.cat(p) for p in zip(*parts)))

    def _extend(self):
        """Where one more token of each sequence goes."""
        n = self.lengths.shape[0]
        if n <= _MOST:
            return self._placing.extend(self.table, self.lengths)
        parts = [self._placing.extend(self.table[i:i + _MOST], self.lengths[i:i + _MOST]) for i in range(0, n, _MOST)]
        return tuple(torch.cat(p) for p in zip(*parts))

    def _forward(self, tokens, positions, slots, attention, keys: bool):
        """Hidden states of `tokens` [n] at `positions`, their keys and values written to `slots`;
        attention(layer, q, k, v) -> [n, heads, dim], k only if it needs the `keys`."""
        c = self.config
        x = self.weights["token_embd.weight"][tokens].float()
        for layer in range(c.layers):
            blk = f"blk.{layer}"
            h = rms_norm(x, self.weights[f"{blk}.attn_norm.weight"], c.eps).bfloat16()
            q, k, v = (self._linear(f"{blk}.attn_{w}", h, torch.bfloat16).unflatten(-1, (n, c.head_dim))
                       for w, n in (("q", c.heads), ("k", c.kv_heads), ("v", c.kv_heads)))
            (q, qw), (k, kw) = self._head_norm(f"{blk}.attn_q_norm.weight", q), self._head_norm(f"{blk}.attn_k_norm.weight", k)
            rows = (q, k, v) if q.dtype == k.dtype == v.dtype else (q.float(), k.float(), v.float())
            q, k = self.caches[layer].append_rotated(*rows, slots, positions, self._inv_freq, qw, kw, c.eps, keys)
            a = attention(layer, q, k, v)
            x = x + self._linear(f"{blk}.attn_output", a.flatten(1))
            h = rms_norm(x, self.weights[f"{blk}.ffn_norm.weight"], c.eps).bfloat16()
            g = torch.nn.functional.silu(self._linear(f"{blk}.ffn_gate", h)) * self._linear(f"{blk}.ffn_up", h)
            x = x + self._linear(f"{blk}.ffn_down", g.bfloat16())
        return x

    def _logits(self, x):
        x = rms_norm(x, self.weights["output_norm.weight"], self.config.eps)
        if "output.weight" in self.weights:
            return self._linear("output", x.bfloat16())
        return x @ self.weights["token_embd.weight"].t()

    @torch.no_grad()
    def prefill(self, prompts: Sequence[Sequence[int]], room: int = 0, beams: int = 1):
        """Start sequences from `prompts` (at least a token each), with pages for `room` more tokens
        of each; returns the logits after each prompt's last token [n, vocab].  With beams, each
        prompt is so many sequences from here on, one after another.  The sequences before
        them end, also where it fails in the middle."""
        lengths = [len(p) for p in prompts]
        if not lengths or min(lengths) == 0:
            raise ValueError("TextDecoder.prefill: at least one prompt, of at least one token each")
        if room < 0 or not 1 <= beams <= MQ_MAX_BEAMS:
            raise ValueError(f"TextDecoder.prefill: room for {room} tokens, {beams} beams")
        if beams > 1:
            if len(lengths) > _MOST:
                raise ValueError(f"TextDecoder.prefill: beams of up to 2^20 prompts, not of {len(lengths)}")
            self._beam_states()
        page = self.page_tokens
        per = -(-(max(lengths) + room) // page)
        shared = [n // page if beams > 1 else 0 for n in lengths]
        need = [s + beams * (-(-(n + room) // page) - s) for s, n in zip(shared, lengths)]
        if sum(need) > self.pages:
            raise ValueError(f"TextDecoder.prefill: {sum(need)} pages needed, the cache has {self.pages}")
        plan = PromptPlan(lengths, self.config.heads, self.config.kv_heads, self.config.head_dim, self.device)
        tokens = torch.tensor([t for p in prompts for t in p])
        vocab = self.weights["token_embd.weight"].shape[0]
        if tokens.min() < 0 or tokens.max() >= vocab:
            raise ValueError(f"TextDecoder.prefill: a token outside 0 .. {vocab - 1}")
        at = self._place(lengths, need, per, room, beams)
        tokens = tokens.to(self.device)
        self._end()
        x = self._forward(tokens, at.positions, at.slots, lambda layer, q, k, v: prompt_attention(q, k, v, plan), keys=True)
        logits = self._logits(x[at.last])
        if beams > 1:                # the partial page of each prompt, of which the first beam has the tokens
            self._beam_states().reorder(at.table, at.lengths, torch.zeros((len(lengths), beams), dtype=torch.int32, device=self.device))
        self._begin(at.table, at.lengths)
        return logits

    def _end(self):
        """The sequences end, their pages are free.  A captured step that still reads their buffers
        finds lengths past the table: it writes nowhere and gives NaN."""
        if self.lengths is not None:
            self.lengths.fill_(self.table.shape[1] * self.page_tokens)
            self._buffers, self.table, self.lengths = (self.table, self.lengths), None, None

    def _begin(self, table, lengths):
        """The sequences to step from here on, in the buffers of those before them if they fit, which a
        captured step reads and writes; buffers that do not fit are kept for such a step."""
        if self._buffers is not None and self._buffers[0].shape == table.shape:
            self.table, self.lengths = self._buffers[0].copy_(table), self._buffers[1].copy_(lengths)
            return
        if self._captured:
            self._retired.append(self._buffers)
            self._captured = False
        self.table, self.lengths = table, lengths

    @torch.no_grad()
    def step(self, tokens):
        """Append `tokens` (int64 [n], on the device, of the vocabulary) to the sequences; returns the
        logits after them.  A sequence past its pages has none left: its logits are NaN."""
        if self.lengths is None:
            raise ValueError("TextDecoder.step: prefill first")
        if tokens.shape != self.lengths.shape or tokens.dtype not in (torch.int64, torch.int32) or tokens.device != self.lengths.device:
            raise ValueError(f"TextDecoder.step: tokens must be int64 {list(self.lengths.shape)} on {self.lengths.device}")
        self._captured |= torch.cuda.is_current_stream_capturing()
        # past the table: written nowhere, and longer than its pages, which attention answers with NaN
        slots, pos, lengths = self._extend()
        x = self._forward(tokens, pos, slots, lambda layer, q, k, v: self.caches[layer].attend(q, self.table, lengths), keys=False)
        logits = self._logits(x)
        self.lengths.copy_(lengths)      # last: a step that fails has not moved the sequences on
        return logits

    def generate(self, prompts: Sequence[Sequence[int]], count: int, stop: Optional[int] = None):
        """The `count` most likely next tokens of each prompt, one after another, [n, count]; a
        sequence repeats `stop` once it has given it."""
        if count < 0:
            raise ValueError(f"TextDecoder.generate: {count} tokens")
        token = self.prefill(prompts, room=count).argmax(-1)
        out = [token]
        for _ in range(count - 1):
            nxt = self.step(token).argmax(-1)
            token = nxt if stop is None else torch.where(token == stop, token, nxt)
            out.append(token)
        return torch.stack(out, 1)[:, :count]

    @torch.no_grad()
    def beam_search(self, prompts: Sequence[Sequence[int]], beams: int, count: int, stop: Optional[int] = None):
        """The continuations of `count` tokens of each prompt that a search with `beams` hypotheses
        finds the most probable, best first -> (tokens [n, beams, count], their log probabilities
        [n, beams]).  A continuation that has given `stop` repeats it and keeps its probability;
        where there are fewer continuations than beams, the rest have tokens -1, probability 0."""
        vocab = self.weights["token_embd.weight"].shape[0]
        if count < 0 or stop is not None and not 0 <= stop < vocab:
            raise ValueError(f"TextDecoder.beam_search: {count} tokens, stop {stop} of {vocab}")
        logits, chosen = self.prefill(prompts, room=count, beams=beams)[:, None], []
        n, last = len(prompts), None
        scores = torch.zeros((n, 1), device=self.device)
        for at in range(count):
            if at:
                logits = self.step(last.clamp(min=0).reshape(-1)).view(n, beams, -1)      # a place left over steps some token
            ended = {} if stop is None or last is None else {"last": last, "stop": stop}
            scores, parents, last = select_beams(logits, scores, beams, **ended)
            if at and beams > 1:
                self._beam_states().reorder(self.table, self.lengths, parents)
            chosen.append((parents, last))
        if not chosen:
            return torch.empty((n, beams, 0), dtype=torch.int64, device=self.device), scores.expand(n, beams).contiguous()
        row, out = torch.arange(beams, device=self.device).expand(n, beams), []
        for parents, tokens in reversed(chosen):
            out.append(torch.gather(tokens, 1, row))
            row = torch.gather(parents.long(), 1, row)
        return torch.where((last < 0)[:, :, None], -1, torch.stack(out[::-1], 2)), scores     # a place left over has no parent
