"""Causal attention of the GGUF text models (the Qwen text encoders, prompt expansion): whole
prompts, and new tokens over a paged key/value cache, run by libmoldq (mq_prompt_attention, mq_kv_cache_* and
mq_cache_attention in include/moldq.h).

candle composes both of matmul, mask and softmax and grows its cache by concatenation
(quantized_qwen3's attention, used at crates/mold-inference/src/expand.rs:200-203).  Here the
prompts of a batch are packed without padding, query heads share k/v heads, and the cache
holds BF16 or the ggml block types Q8_0 and Q4_0.

Everything runs on torch's current stream of the tensors' device and allocates only outputs
and scratch.  Inference only: calls that autograd or a tracer would record are refused.
"""
from __future__ import annotations

import ctypes

import numpy as np
import torch

from . import _lib
from ._lib import check
from .fused import recorded
from .quantized import GgmlDType, _dtype_code

_MAX_STRIDE = 1 << 24
_BF16 = torch.bfloat16


class _OnStreams:
    """Device memory that an object keeps for its calls, told to the allocator for each stream that
    they run on: memory of an object that is dropped is given out again only after them."""

    def __init__(self, t):
        self.t, self.device = t, t.device
        self.streams = {torch._C._cuda_getCurrentRawStream(t.device.index)}

    def run(self, fn, *args):
        """fn(*args, torch's current stream) with the device current, as it mostly is (making it so
        takes 1.3 us of a 9 us call)."""
        current = torch._C._cuda_getDevice()
        if current != self.device.index:
            with torch.cuda.device(self.device):
                return self.run(fn, *args)
        stream = torch._C._cuda_getCurrentRawStream(current)
        if stream not in self.streams:
            self.t.record_stream(torch.cuda.current_stream())
            self.streams.add(stream)
        rc = fn(*args, stream)
        if rc:
            check(rc)


def _operand(name, t, shape, device):
    """t as the library reads it, with its token and head stride: bf16 `shape` = (tokens, heads,
    dim) on `device`; copied unless it has unit stride along the head and 16-byte rows."""
    if t.dtype is not _BF16 or t.shape != shape or t.device != device:
        raise ValueError(f"{name} must be bf16 {list(shape)} on {device}")
    st, sh, sd = t.stride()
    if sd != 1 or (st | sh) & 7 or st >= _MAX_STRIDE or sh >= _MAX_STRIDE or t.data_ptr() & 15:
        if not _readable(t):
            t = _copied(t)
        st, sh = _strides(t)
    return t, st, sh


def _copied(t):
    """t's values packed and aligned; contiguous() would return a packed t as it is, off 16 bytes too."""
    return t.clone(memory_format=torch.contiguous_format)


def _readable(t):
    st, sh, sd = t.stride()
    n, h, _ = t.shape
    return (sd == 1 and t.data_ptr() % 16 == 0 and (n <= 1 or (st % 8 == 0 and st < _MAX_STRIDE))
            and (h == 1 or (sh % 8 == 0 and sh < _MAX_STRIDE)))


def _strides(t):
    """Token and head stride; those of a single token or head, which may be anything, as if packed."""
    n, h, d = t.shape
    sh = t.stride(1) if h > 1 else d
    return (t.stride(0) if n > 1 else h * d), sh


def _writable(t):
    """Whether the kernels can store into t as it is: readable, with rows and heads apart."""
    if not _readable(t):
        return False
    n, h, d = t.shape
    st, sh = _strides(t)
    if n == 1 or h == 1:
        return (n == 1 or st >= d) and (h == 1 or sh >= d)
    return st >= d and sh >= d and (st >= (h - 1) * sh + d or sh >= (n - 1) * st + d)


def _span(t):
    """The addresses from t's first byte to past its last."""
    last = sum((n - 1) * stride for n, stride in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _apart(out, t):
    if out.untyped_storage().data_ptr() != t.untyped_storage().data_ptr():
        return True
    (lo, hi), (a, b) = _span(out), _span(t)
    return b <= lo or hi <= a


def _out(name, out, shape, device, inputs):
    """The tensor to write and its strides: `out`, or a temporary where the kernel cannot store
    into it (another device, unaligned or overlapping rows, over an input that other workgroups
    still read)."""
    if out is not None:
        if out.dtype is not _BF16 or out.shape != shape:
            raise ValueError(f"{name}: out must be bf16 {list(shape)}")
        if out.device == device and (out.is_contiguous() and not out.data_ptr() & 15 or _writable(out)):
            for t in inputs:
                if not _apart(out, t):
                    break
            else:
                return out, *_strides(out)
    return inputs[0].new_empty(shape), shape[1] * shape[2], shape[2]


def _given(out, res):
    if out is None:
        return res
    if res is out:
        torch.autograd.graph.increment_version(out)     # written in place, as a copy_ tells autograd
        return out
    return out.copy_(res)


class PromptPlan:
    """How a batch of packed prompts is attended, made once for its lengths and used by every
    layer with these heads: prompt s is the `lengths[s]` rows after those of the prompts before
    it.  heads a multiple of kv_heads, head_dim 64 or 128."""

    def __init__(self, lengths, heads: int, kv_heads: int, head_dim: int = 128, device="cuda"):
        self.lengths = [int(x) for x in lengths]
        lib = _lib.load()
        host = (ctypes.c_int64 * max(1, len(self.lengths)))(*self.lengths)
        self.c = _lib.PromptPlanC()
        args = (host, len(self.lengths), int(heads), int(kv_heads), int(head_dim), ctypes.byref(self.c))
        check(lib.mq_prompt_plan_make(*args, None, 0))
        tiles = np.zeros((max(1, self.c.tiles), 4), dtype=np.int32)
        check(lib.mq_prompt_plan_make(*args, tiles.ctypes.data_as(ctypes.POINTER(ctypes.c_int32)), len(tiles)))
        self.tiles = torch.from_numpy(tiles).to(device)
        self.device = self.tiles.device
        if self.device.type != "cuda":
            raise ValueError(f"PromptPlan: a GPU's, not {self.device}")
        self.tokens = int(self.c.tokens)
        self.heads, self.kv_heads, self.head_dim = int(heads), int(kv_heads), int(head_dim)
        self.q_shape = (self.tokens, self.heads, self.head_dim)
        self.kv_shape = (self.tokens, self.kv_heads, self.head_dim)
        self._ref, self._tiles = ctypes.byref(self.c), self.tiles.data_ptr()
        self._run = _OnStreams(self.tiles).run


def prompt_attention(q, k, v, plan: PromptPlan, scale=None, out=None):
    """Causal attention inside each of the plan's prompts: q bf16 [tokens, heads, dim], k and v
    bf16 [tokens, kv_heads, dim] (views of one projection's output are read in place) ->
    bf16 [tokens, heads, dim], `out` if given.  scale defaults to dim ** -0.5."""
    device, n = plan.device, plan.tokens
    if recorded(q, k, v) if out is None else recorded(q, k, v, out):
        raise ValueError("prompt_attention: inference only, nothing may record the call")
    q, qt, qh = _operand("prompt_attention: q", q, plan.q_shape, device)
    k, kt, kh = _operand("prompt_attention: k", k, plan.kv_shape, device)
    v, vt, vh = _operand("prompt_attention: v", v, plan.kv_shape, device)
    res, ot, oh = _out("prompt_attention", out, plan.q_shape, device, (q, k, v))
    if n:
        plan._run(_lib.load().mq_prompt_attention, plan._ref, plan._tiles, q.data_ptr(), qt, qh, k.data_ptr(), kt, kh,
                  v.data_ptr(), vt, vh, plan.head_dim ** -0.5 if scale is None else scale, res.data_ptr(), ot, oh)
    return _given(out, res)


class KvCache:
    """A paged key/value cache on the device, of `pages` pages of `page_tokens` tokens (a multiple
    of 32), BF16 or in Q8_0 / Q4_0 blocks along the head; head_dim 64 or 128.  Slot s is token
    s % page_tokens of page s // page_tokens; which pages a sequence has is the caller's page table."""

    def __init__(self, pages: int, kv_heads: int, head_dim: int = 128, page_tokens: int = 64,
                 dtype: GgmlDType = GgmlDType.Q8_0, device="cuda"):
        self.c = _lib.KvCacheC(None, int(pages), int(dtype), int(kv_heads), int(head_dim), int(page_tokens))
        self._ref = ctypes.byref(self.c)
        lib = _lib.load()
        size = lib.mq_kv_cache_size(self._ref)
        if size == 0 and pages != 0:
            raise ValueError("KvCache: BF16, Q8_0 or Q4_0, heads of 64 or 128, pages of a multiple of 32 tokens up to 65536, "
                             f"1 to 4096 heads, less than 2^63 bytes; got {GgmlDType(dtype).name}, {head_dim}, {page_tokens}, "
                             f"{kv_heads}, {pages} pages")
        self.data = torch.empty(size, dtype=torch.uint8, device=device)
        self.c.data = self.data.data_ptr()
        self.device = self.data.device
        if self.device.type != "cuda":
            raise ValueError(f"KvCache: a GPU's, not {self.device}")
        self.pages, self.kv_heads, self.head_dim, self.page_tokens = int(pages), int(kv_heads), int(head_dim), int(page_tokens)
        self.dtype = GgmlDType(dtype)
        self._run = _OnStreams(self.data).run

    def slots(self, page_table, positions):
        """The slots of `positions` [batch, n] of the sequences whose pages are page_table
        [batch, pages]; -1 (skipped by append) for a negative position and one past the table."""
        at = positions.clamp(min=0).long()
        column, pages = at // self.page_tokens, page_table.shape[1]
        if pages == 0:
            return torch.full_like(at, -1)
        page = torch.gather(page_table.long(), 1, column.clamp(max=pages - 1))
        return torch.where((positions < 0) | (column >= pages), -1, page * self.page_tokens + at % self.page_tokens)

    def _slots(self, name, slots):
        if slots.dtype is not torch.int64 or slots.dim() != 1 or slots.device != self.device:
            raise ValueError(f"{name}: slots must be int64 [tokens] on {self.device}")
        return slots if slots.is_contiguous() else slots.contiguous()

    def append(self, k, v, slots):
        """Write k and v [tokens, kv_heads, head_dim] (bf16 or f32, both the same) to `slots`, int64
        [tokens] on the device; a slot outside the cache is skipped.  Two tokens must not share one."""
        if recorded(k, v):
            raise ValueError("KvCache.append: inference only, nothing may record the call")
        slots = self._slots("KvCache.append", slots)
        n = slots.shape[0]
        shape, dtype = (n, self.kv_heads, self.head_dim), k.dtype
        if dtype not in (_BF16, torch.float32):
            raise ValueError("KvCache.append: k and v must be bf16 or f32")
        k, kt, kh = self._rows(k, shape, dtype)
        v, vt, vh = self._rows(v, shape, dtype)
        if n:
            self._run(_lib.load().mq_kv_cache_append, self._ref, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh,
                      _dtype_code(dtype), n, slots.data_ptr())

    def _rows(self, t, shape, dtype):
        if t.dtype is not dtype or t.shape != shape or t.device != self.device:
            raise ValueError(f"KvCache.append: k and v must be {list(shape)} of one type on {self.device}")
        st, sh, sd = t.stride()
        mask = 7 if dtype is _BF16 else 3
        if sd != 1 or (st | sh) & mask or st >= _MAX_STRIDE or sh >= _MAX_STRIDE or t.data_ptr() & 15:
            st, sh = _strides(t)
            if sd != 1 or (st | sh) & mask or st >= _MAX_STRIDE or sh >= _MAX_STRIDE or t.data_ptr() & 15:
                t = _copied(t)
                st, sh = _strides(t)
        return t, st, sh

    def read(self, slots, dtype=torch.bfloat16):
        """(k, v) [tokens, kv_heads, head_dim] of `slots`, bf16 or f32; zeros for a slot outside the cache."""
        if recorded(slots):
            raise ValueError("KvCache.read: inference only, nothing may record the call")
        slots = self._slots("KvCache.read", slots)
        if dtype not in (torch.bfloat16, torch.float32):
            raise ValueError("KvCache.read: dtype must be bf16 or f32")
        shape = (slots.shape[0], self.kv_heads, self.head_dim)
        k = torch.empty(shape, dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        if shape[0]:
            self._run(_lib.load().mq_kv_cache_read, self._ref, slots.data_ptr(), shape[0], k.data_ptr(), v.data_ptr(),
                      _dtype_code(dtype))
        return k, v

    def attend(self, q, page_table, lengths, scale=None, out=None):
        """Attention of one new token per sequence: q bf16 [batch, heads, head_dim] over the first
        lengths[b] tokens (int32 [batch], the new one's included once it is appended) of the pages
        page_table[b] (int32 [batch, pages]) -> bf16 [batch, heads, head_dim], `out` if given.
        scale defaults to head_dim ** -0.5.  Table and lengths are read on the device."""
        device, dim = self.device, self.head_dim
        if recorded(q) if out is None else recorded(q, out):
            raise ValueError("KvCache.attend: inference only, nothing may record the call")
        if q.dim() != 3 or q.shape[1] == 0 or q.shape[1] % self.kv_heads:
            raise ValueError(f"KvCache.attend: q must be [batch, heads, {dim}] with a multiple of {self.kv_heads} heads")
        n, heads, _ = q.shape
        q, qb, qh = _operand("KvCache.attend: q", q, (n, heads, dim), device)
        for name, t, dims in (("page_table", page_table, 2), ("lengths", lengths, 1)):
            if t.dtype is not torch.int32 or t.dim() != dims or t.shape[0] != n or t.device != device:
                raise ValueError(f"KvCache.attend: {name} must be int32 [{n}{', pages' if dims == 2 else ''}] on {device}")
        pages = page_table.shape[1]
        if n > 1 and page_table.stride(0) < pages or pages > 1 and page_table.stride(1) != 1:
            page_table = page_table.contiguous()
        if not lengths.is_contiguous():
            lengths = lengths.contiguous()
        res, ob, oh = _out("KvCache.attend", out, (n, heads, dim), device, (q,))
        if n:
            lib = _lib.load()
            nbytes = lib.mq_cache_attention_scratch_size(self._ref, n, heads, pages)
            scratch = self.data.new_empty(nbytes) if nbytes else None     # freed to this stream
            self._run(lib.mq_cache_attention, self._ref, q.data_ptr(), qb, qh, n, heads, page_table.data_ptr(),
                      page_table.stride(0) if n > 1 else pages, pages, lengths.data_ptr(),
                      dim ** -0.5 if scale is None else scale, res.data_ptr(), ob, oh, scratch.data_ptr() if nbytes else None,
                      nbytes)
        return _given(out, res)
