"""A GGUF text decoder on the library's linears and text attention: prompts in, tokens out.

What mold's prompt expansion runs through candle's quantized_qwen3::ModelWeights
(crates/mold-inference/src/expand.rs:200-203): RmsNorm, grouped-head attention with rotary
halves and optional q/k head norms, and a SwiGLU MLP, with tensor names as GGUF files give
them (TextConfig.from_metadata and gguf.Content.var_builder make one of a file).  `prefill`
takes a batch of prompts packed without padding, `step` one new token of each sequence; both
write their keys and values into one paged cache (quantized where its type is a block type)
that `step` attends over.  Norms, rotations and the activation are torch operations in float32;
projections are QMatMul, attention and cache text_attention.

`step` makes no host synchronization: lengths and page table stay on the device, so it can be
captured in a graph.  The graph goes on to a later prefill's sequences if there are as many and
their page table is as wide; otherwise its replays write nothing and give NaN, and a step has to
be captured anew.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, Optional, Sequence

import torch

from .quantized import GgmlDType, QMatMul, QTensor
from .text_attention import KvCache, PromptPlan, prompt_attention


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
    """Rotary embedding of the halves of each head: x [tokens, heads, dim], cos and sin [tokens, dim / 2]."""
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
        self.table = self.lengths = self._buffers = None
        self._captured, self._retired = False, []     # what graphs of earlier batches hold
        half = config.head_dim // 2
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

    def _heads(self, blk: str, which: str, x, heads: int, cos, sin):
        y = self._linear(f"{blk}.attn_{which}", x, torch.bfloat16).unflatten(-1, (heads, self.config.head_dim))
        if which == "v":
            return y
        weight = self.weights.get(f"{blk}.attn_{which}_norm.weight")
        if weight is not None:
            y = rms_norm(y, weight, self.config.eps)
        return rotate(y, cos, sin).bfloat16()

    def _forward(self, tokens, positions, slots, attention):
        """Hidden states of `tokens` [n] at `positions`, their keys and values written to `slots`;
        attention(layer, q, k, v) -> [n, heads, dim]."""
        c = self.config
        angle = positions.float()[:, None] * self._inv_freq
        cos, sin = angle.cos(), angle.sin()
        x = self.weights["token_embd.weight"][tokens].float()
        for layer in range(c.layers):
            blk = f"blk.{layer}"
            h = rms_norm(x, self.weights[f"{blk}.attn_norm.weight"], c.eps).bfloat16()
            q, k, v = (self._heads(blk, w, h, n, cos, sin) for w, n in (("q", c.heads), ("k", c.kv_heads), ("v", c.kv_heads)))
            self.caches[layer].append(k, v, slots)
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
    def prefill(self, prompts: Sequence[Sequence[int]], room: int = 0):
        """Start sequences from `prompts` (at least a token each), with pages for `room` more tokens
        of each; returns the logits after each prompt's last token [n, vocab].  The sequences before
        them end, also where it fails in the middle."""
        lengths = [len(p) for p in prompts]
        if not lengths or min(lengths) == 0:
            raise ValueError("TextDecoder.prefill: at least one prompt, of at least one token each")
        if room < 0:
            raise ValueError(f"TextDecoder.prefill: room for {room} tokens")
        per = -(-(max(lengths) + room) // self.page_tokens)
        need = [-(-(n + room) // self.page_tokens) for n in lengths]
        if sum(need) > self.pages:
            raise ValueError(f"TextDecoder.prefill: {sum(need)} pages needed, the cache has {self.pages}")
        table, at = torch.full((len(lengths), per), -1, dtype=torch.int32), 0
        for b, n in enumerate(need):
            table[b, :n] = torch.arange(at, at + n)
            at += n
        pos = torch.cat([torch.arange(n) for n in lengths])
        seq = torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(lengths))
        slots = table.long()[seq, pos // self.page_tokens] * self.page_tokens + pos % self.page_tokens
        slots, pos = slots.to(self.device), pos.to(self.device)
        plan = PromptPlan(lengths, self.config.heads, self.config.kv_heads, self.config.head_dim, self.device)
        tokens = torch.tensor([t for p in prompts for t in p])
        vocab = self.weights["token_embd.weight"].shape[0]
        if tokens.min() < 0 or tokens.max() >= vocab:
            raise ValueError(f"TextDecoder.prefill: a token outside 0 .. {vocab - 1}")
        tokens = tokens.to(self.device)
        last = torch.cumsum(torch.tensor(lengths), 0) - 1
        self._end()
        x = self._forward(tokens, pos, slots, lambda layer, q, k, v: prompt_attention(q, k, v, plan))
        logits = self._logits(x[last.to(self.device)])
        self._begin(table, torch.tensor(lengths, dtype=torch.int32))
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
        self.table, self.lengths = table.to(self.device), lengths.to(self.device)

    @torch.no_grad()
    def step(self, tokens):
        """Append `tokens` (int64 [n], on the device, of the vocabulary) to the sequences; returns the
        logits after them.  A sequence past its pages has none left: its logits are NaN."""
        if self.lengths is None:
            raise ValueError("TextDecoder.step: prefill first")
        if tokens.shape != self.lengths.shape or tokens.dtype not in (torch.int64, torch.int32) or tokens.device != self.lengths.device:
            raise ValueError(f"TextDecoder.step: tokens must be int64 {list(self.lengths.shape)} on {self.lengths.device}")
        self._captured |= torch.cuda.is_current_stream_capturing()
        pos, lengths = self.lengths.long(), self.lengths + 1
        held = torch.full_like(pos, self.table.shape[1] * self.page_tokens)
        # past the table: written nowhere, and longer than its pages, which attention answers with NaN
        slots = torch.where(pos < held, self.caches[0].slots(self.table, torch.minimum(pos, held - 1)[:, None])[:, 0], -1)
        x = self._forward(tokens, pos, slots, lambda layer, q, k, v: self.caches[layer].attend(q, self.table, lengths))
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
