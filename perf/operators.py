"""Text attention: the workloads its operators are timed on, and their plain forms.

`prompt`: causal attention with grouped heads over packed prompts of different lengths.
`cache`: keys and values written into the paged cache (quantized on the way, where its type is
a block type) and read back.
`decode`: attention of one new token per sequence over that cache.

`own` False computes each operator with elementary torch operations in float32; True calls
mold_amd.text_attention.  Inputs are made on the GPU from the seed; lengths come from the case.
"""
import math
import random
import zlib

import torch

own = False

BLOCK = 32                                                   # values of a quantized block, along the head
BYTES = {"bf16": 2.0, "q8_0": 34 / BLOCK, "q4_0": 18 / BLOCK}   # a stored value
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # a text encoder's prompt of 77 tokens, as many key as query heads, heads of 64: the launch is the cost
        {"name": "prompt_77", "op": "prompt", "heads": 12, "kv": 12, "dim": 64, "n": 1, "longest": 77, "mix": 0},
        # one prompt to expand, grouped heads
        {"name": "prompt_500", "op": "prompt", "heads": 16, "kv": 8, "dim": 128, "n": 1, "longest": 500, "mix": 0},
        # prompts of a batch packed one after another, odd lengths, the shortest of a token or so
        {"name": "prompt_packed", "op": "prompt", "heads": 32, "kv": 8, "dim": 128, "n": 24, "longest": 1000, "mix": 1},
        # a long document
        {"name": "prompt_8192", "op": "prompt", "heads": 32, "kv": 8, "dim": 128, "n": 1, "longest": 8192, "mix": 0},
        # one decode step's tokens, written and read back: the launches are the cost
        {"name": "cache_step", "op": "cache", "kv": 8, "dim": 128, "tokens": 48, "type": "q8_0", "input": "bf16", "page": 64},
        # a prompt's keys and values straight from f32 linears
        {"name": "cache_prompt", "op": "cache", "kv": 8, "dim": 128, "tokens": 4100, "type": "q8_0", "input": "f32", "page": 64},
        # a batch of long prompts into the smallest type
        {"name": "cache_long_q4", "op": "cache", "kv": 8, "dim": 128, "tokens": 32768, "type": "q4_0", "input": "bf16", "page": 128},
        # one sequence a few hundred tokens on
        {"name": "decode_one", "op": "decode", "heads": 16, "kv": 8, "dim": 128, "n": 1, "longest": 700, "mix": 0, "type": "q8_0", "page": 64},
        # one sequence over a long context: only a split over its length fills the card
        {"name": "decode_one_long", "op": "decode", "heads": 32, "kv": 8, "dim": 128, "n": 1, "longest": 65001, "mix": 0, "type": "bf16", "page": 64},
        # a serving batch of sequences of all ages
        {"name": "decode_ragged", "op": "decode", "heads": 32, "kv": 8, "dim": 128, "n": 40, "longest": 6000, "mix": 2, "type": "q8_0", "page": 32},
        # heads of 64 without groups, the smallest type
        {"name": "decode_q4_heads64", "op": "decode", "heads": 20, "kv": 20, "dim": 64, "n": 16, "longest": 3500, "mix": 3, "type": "q4_0", "page": 64},
        # the largest: a full batch at a long context
        {"name": "decode_full", "op": "decode", "heads": 32, "kv": 8, "dim": 128, "n": 64, "longest": 8192, "mix": 0, "type": "bf16", "page": 128},
    ]


def _between(rng, lo, hi):
    """A whole number, spread over its logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    heads, kv = rng.choice([(12, 12), (16, 8), (32, 8), (20, 20), (8, 1), (28, 4), (24, 8), (16, 2), (40, 8)])
    c = {"heads": heads, "kv": kv, "dim": rng.choice([64, 128, 128])}
    op = rng.choice(["prompt", "cache", "decode"])
    c["op"] = op
    if op == "prompt":
        n = _between(rng, 1, 32)
        longest = _between(rng, 1, min(6000, int(math.sqrt(32e6 / n))))    # n x longest^2 below the largest listed case's
        return {**c, "n": n, "longest": longest, "mix": rng.randrange(0, 1000)}
    c["type"] = rng.choice(["bf16", "q8_0", "q4_0"])
    c["page"] = rng.choice([32, 64, 96, 128, 256])
    if op == "cache":
        del c["heads"]
        return {**c, "tokens": _between(rng, 1, 160000 // kv), "input": rng.choice(["bf16", "f32"])}
    n = _between(rng, 1, 64)
    return {**c, "n": n, "longest": _between(rng, 1, min(65536, 3000000 // (n * kv))), "mix": rng.randrange(0, 1000)}


def _lengths(case):
    """The sequences' lengths: all the longest for mix 0, else spread below it, the longest among them."""
    n, longest, mix = case["n"], case["longest"], case["mix"]
    if mix == 0:
        return [longest] * n
    rng = random.Random(mix)
    return [longest] + [_between(rng, 1, longest) if k % 2 else rng.randint(1, longest) for k in range(1, n)]


def _gen(seed, name):
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(f"{seed}/{name}".encode()))


def _rows(seed, name, *shape, dtype=torch.bfloat16):
    """N(0, 1) values whose channels differ in size by a factor of a few, as projections give them."""
    g = _gen(seed, name)
    size = torch.exp(0.4 * torch.randn(shape[-1], device="cuda", generator=g))
    return (torch.randn(shape, device="cuda", generator=g) * size).to(dtype)


def _text():
    from mold_amd import text_attention
    return text_attention


def _cache(case, pages):
    from mold_amd import GgmlDType
    kind = {"bf16": GgmlDType.BF16, "q8_0": GgmlDType.Q8_0, "q4_0": GgmlDType.Q4_0}[case["type"]]
    return _text().KvCache(pages, case["kv"], case["dim"], page_tokens=case["page"], dtype=kind, device="cuda")


# ------------------------------------------------------------------ inputs

def prepare(case, seed):
    return {"prompt": _prepare_prompt, "cache": _prepare_cache, "decode": _prepare_decode}[case["op"]](case, seed)


def _prepare_prompt(case, seed):
    lengths = _lengths(case)
    total, h, kv, d = sum(lengths), case["heads"], case["kv"], case["dim"]
    qkv = _rows(seed, "qkv", total, h + 2 * kv, d)               # one projection's output, its parts side by side
    state = {"op": "prompt", "q": qkv[:, :h], "k": qkv[:, h:h + kv], "v": qkv[:, h + kv:], "scale": d ** -0.5}
    if own:
        state["plan"] = _text().PromptPlan(lengths, h, kv, d, device="cuda")
        return state
    # the padded form's indices: which packed row each (prompt, position) is, and where each packed row sits
    n, longest = len(lengths), max(lengths)
    size = torch.tensor(lengths, device="cuda")
    start = torch.cumsum(size, 0) - size
    pos = torch.arange(longest, device="cuda")
    state["gather"] = (start[:, None] + torch.minimum(pos[None], size[:, None] - 1)).reshape(-1)
    state["back"] = torch.nonzero((pos[None] < size[:, None]).reshape(-1)).reshape(-1)
    state["n"], state["longest"] = n, longest
    return state


def _slots(case, seed, tokens):
    """Pages of the pool in no order, and the slot of each token in them."""
    page = case["page"]
    used = -(-tokens // page)
    pool = used + 3
    order = torch.randperm(pool, device="cuda", generator=_gen(seed, "pages"))[:used]
    t = torch.arange(tokens, device="cuda")
    return pool, order, order[t // page] * page + t % page


def _prepare_cache(case, seed):
    t, kv, d = case["tokens"], case["kv"], case["dim"]
    kvs = _rows(seed, "kv", t, 2 * kv, d, dtype=DTYPES[case["input"]])
    pool, _, slots = _slots(case, seed, t)
    state = {"op": "cache", "type": case["type"], "k": kvs[:, :kv], "v": kvs[:, kv:], "slots": slots}
    if own:
        state["cache"] = _cache(case, pool)
    else:
        state["cache"] = _plain_pool(case["type"], pool * case["page"], kv, d)
    return state


def _prepare_decode(case, seed):
    lengths = _lengths(case)
    h, kv, d, page = case["heads"], case["kv"], case["dim"], case["page"]
    per = [-(-x // page) for x in lengths]
    width = max(per) + 1
    used = sum(per)
    order = torch.randperm(used + 3, device="cuda", generator=_gen(seed, "pages")).to(torch.int32)
    table = torch.zeros((len(lengths), width), dtype=torch.int32, device="cuda")
    held = torch.arange(width, device="cuda")[None] < torch.tensor(per, device="cuda")[:, None]
    table[held] = order[:used]
    state = {"op": "decode", "type": case["type"], "q": _rows(seed, "q", len(lengths), h, d), "table": table,
             "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"), "scale": d ** -0.5, "page": page}
    slots = torch.arange((used + 3) * page, device="cuda")
    k, v = _history(case, seed, (used + 3) * page)
    if own:
        state["cache"] = _cache(case, used + 3)
        state["cache"].append(k, v, slots)
    else:
        state["cache"] = _plain_pool(case["type"], (used + 3) * page, kv, d)
        _plain_append(case["type"], state["cache"], k, v, slots)
    return state


def _history(case, seed, slots):
    """What the whole pool holds before the step, slot by slot."""
    return (_rows(seed, "hk", slots, case["kv"], case["dim"]), _rows(seed, "hv", slots, case["kv"], case["dim"]))


# ------------------------------------------------------------------ plain forms

def _plain_pool(kind, slots, kv, d):
    """A cache as plain tensors, keys first: values, or whole numbers and the scale of each block."""
    if kind == "bf16":
        return {"x": torch.zeros((2, slots, kv, d), dtype=torch.bfloat16, device="cuda")}
    return {"x": torch.zeros((2, slots, kv, d), dtype=torch.int8, device="cuda"),
            "d": torch.zeros((2, slots, kv, d // BLOCK), dtype=torch.float16, device="cuda")}


def _plain_blocks(kind, x):
    """Whole numbers and float16 scales of x's blocks of 32."""
    b = x.float().unflatten(-1, (-1, BLOCK))
    if kind == "q8_0":
        d = b.abs().amax(-1, keepdim=True) / 127.0
        inv = torch.where(d != 0, 1.0 / d, torch.zeros_like(d))
        y = b * inv
        q = torch.trunc(y + torch.copysign(torch.full_like(y, 0.5), y))      # halves away from zero
        # 0.5 added to the float below one half rounds up to 1
        q = torch.where(y.abs() < 0.5, torch.zeros_like(q), q)
    else:
        first = torch.argmax(b.abs(), dim=-1, keepdim=True)
        d = torch.gather(b, -1, first) / -8.0
        inv = torch.where(d != 0, 1.0 / d, torch.zeros_like(d))
        q = torch.clamp(torch.trunc(b * inv + 8.5), max=15.0) - 8.0
    return q.flatten(-2).to(torch.int8), d.squeeze(-1).half()


def _plain_append(kind, pool, k, v, slots):
    kv = torch.stack([k, v])
    if kind == "bf16":
        pool["x"][:, slots] = kv.bfloat16()
        return
    q, d = _plain_blocks(kind, kv)
    pool["x"][:, slots] = q
    pool["d"][:, slots] = d


def _plain_values(kind, pool, slots):
    """float32 [2, .., kv, d] of the slots."""
    x = pool["x"][:, slots].float()
    if kind == "bf16":
        return x
    return (x.unflatten(-1, (-1, BLOCK)) * pool["d"][:, slots].float().unsqueeze(-1)).flatten(-2)


def _plain_prompt(s):
    n, longest = s["n"], s["longest"]
    q, k, v = (s[x][s["gather"]].float().unflatten(0, (n, longest)).permute(0, 2, 1, 3).contiguous() for x in "qkv")
    heads, kv, d = q.shape[1], k.shape[1], q.shape[3]
    q = q.reshape(n, kv, heads // kv * longest, d)                           # a group's rows beside each other
    w = torch.matmul(q, k.transpose(2, 3)).mul_(s["scale"]).reshape(n, heads, longest, longest)
    pos = torch.arange(longest, device="cuda")
    w.masked_fill_(pos[None, :] > pos[:, None], -math.inf)
    w.sub_(w.amax(-1, keepdim=True)).exp_()
    total = w.sum(-1, keepdim=True)
    o = torch.matmul(w.reshape(n, kv, heads // kv * longest, longest), v).reshape(n, heads, longest, d) / total
    return o.permute(0, 2, 1, 3).reshape(n * longest, heads, d)[s["back"]].bfloat16()


def _plain_decode(s):
    n, width = s["table"].shape
    heads, d = s["q"].shape[1:]
    page = s["page"]
    pos = torch.arange(width * page, device="cuda")
    slots = s["table"].long()[:, pos // page] * page + pos % page
    k, v = _plain_values(s["type"], s["cache"], slots)                       # [n, positions, kv, d]
    kv = k.shape[2]
    q = s["q"].float().reshape(n, kv, heads // kv, d)
    w = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()).mul_(s["scale"])
    w.masked_fill_((pos[None] >= s["lengths"][:, None])[:, None, None], -math.inf)
    w.sub_(w.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(w, v.transpose(1, 2).contiguous()) / w.sum(-1, keepdim=True)
    return o.reshape(n, heads, d).bfloat16()


def run(state):
    op = state["op"]
    if op == "prompt":
        if own:
            return _text().prompt_attention(state["q"], state["k"], state["v"], state["plan"], scale=state["scale"])
        return _plain_prompt(state)
    if op == "cache":
        if own:
            state["cache"].append(state["k"], state["v"], state["slots"])
            return state["cache"].read(state["slots"], dtype=torch.bfloat16)
        _plain_append(state["type"], state["cache"], state["k"], state["v"], state["slots"])
        k, v = _plain_values(state["type"], state["cache"], state["slots"]).bfloat16()
        return k, v
    if own:
        return state["cache"].attend(state["q"], state["table"], state["lengths"], scale=state["scale"])
    return _plain_decode(state)


# ------------------------------------------------------------------ what a pass needs

def work(case):
    kv, d = case["kv"], case["dim"]
    if case["op"] == "cache":
        values = 2 * case["tokens"] * kv * d
        size = 4 if case["input"] == "f32" else 2
        return {"bytes": values * (size + 2 * BYTES[case["type"]] + 2) + 16 * case["tokens"], "flops": 4 * values}
    lengths, h = _lengths(case), case["heads"]
    if case["op"] == "prompt":
        return {"bytes": 2 * d * sum(lengths) * (2 * h + 2 * kv), "flops": 4 * d * h * sum(x * (x + 1) // 2 for x in lengths)}
    return {"bytes": 2 * d * kv * sum(lengths) * BYTES[case["type"]] + 4 * d * h * len(lengths), "flops": 4 * d * h * sum(lengths)}


# ------------------------------------------------------------------ 64 bits

def _exact_blocks(kind, x):
    """The values that x's quantized blocks stand for, by the definition."""
    shape = x.shape
    b = x.double().reshape(-1, BLOCK)
    if kind == "q8_0":
        d = b.abs().max(1, keepdim=True).values / 127
        q = torch.where(d > 0, (b.abs() / d.clamp(min=1e-300) + 0.5).floor() * b.sign(), torch.zeros_like(b))
    else:
        i = b.abs().max(1, keepdim=True)
        # the first value of the largest magnitude
        at = (b.abs() == i.values).to(torch.int8).argmax(1, keepdim=True)
        d = -torch.take_along_dim(b, at, 1) / 8
        q = torch.where(d != 0, (b / torch.where(d != 0, d, torch.ones_like(d)) + 8.5).floor().clamp(max=15) - 8, torch.zeros_like(b))
    return (q * d.half().double()).reshape(shape)


def _stored(kind, x):
    return x.to(torch.bfloat16).double() if kind == "bf16" else _exact_blocks(kind, x)


def _softmax64(q, k, v, scale, causal):
    """q [rows, d], k and v [keys, d]: the rows' attention, row i over keys 0 .. i + keys - rows where causal."""
    s = (q @ k.t()) * scale
    if causal:
        s = s + torch.full_like(s, -math.inf).triu(1 + k.shape[0] - q.shape[0])
    return torch.softmax(s, -1) @ v


def exact(case, seed):
    kv, d = case["kv"], case["dim"]
    if case["op"] == "cache":
        kvs = _rows(seed, "kv", case["tokens"], 2 * kv, d, dtype=DTYPES[case["input"]])
        x = _stored(case["type"], kvs)
        return x[:, :kv].contiguous(), x[:, kv:].contiguous()
    lengths, h = _lengths(case), case["heads"]
    group = h // kv
    if case["op"] == "prompt":
        qkv = _rows(seed, "qkv", sum(lengths), h + 2 * kv, d).double()
        out, at = torch.empty((sum(lengths), h, d), dtype=torch.float64, device="cuda"), 0
        for x in lengths:
            for i in range(h):
                rows = qkv[at:at + x]
                out[at:at + x, i] = _softmax64(rows[:, i], rows[:, h + i // group], rows[:, h + kv + i // group], d ** -0.5, True)
            at += x
        return out
    page = case["page"]
    per = [-(-x // page) for x in lengths]
    order = torch.randperm(sum(per) + 3, device="cuda", generator=_gen(seed, "pages"))
    hk, hv = _history(case, seed, (sum(per) + 3) * page)
    q = _rows(seed, "q", len(lengths), h, d).double()
    out, at = torch.empty((len(lengths), h, d), dtype=torch.float64, device="cuda"), 0
    for b, x in enumerate(lengths):
        slots = (order[at:at + per[b], None] * page + torch.arange(page, device="cuda")).reshape(-1)[:x]
        k, v = _stored(case["type"], hk[slots]), _stored(case["type"], hv[slots])
        for i in range(kv):
            out[b, i * group:(i + 1) * group] = _softmax64(q[b, i * group:(i + 1) * group], k[:, i], v[:, i], d ** -0.5, False)
        at += per[b]
    return out
