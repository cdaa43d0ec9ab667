"""The text decoder's steps between its linears and its attention, and beam search: the workloads
their operators are timed on, and their plain forms.

`heads`: q and k of each head normed and rotated to their positions; with a cache, k and v also
written into it and read back.
`place`: page table, slots and positions of packed prompts, or of sequences that go on, made on
the GPU from their lengths.
`select`: the best continuations of each request's beams over the whole vocabulary.
`reorder`: the beams' page tables by their parents, shared partial pages copied in every layer.

`own` False computes each operator with elementary torch operations; True calls
mold_amd.text_attention and mold_amd.beams.  Inputs are made on the GPU from the seed; lengths and
parents come from the case.
"""
import math
import random
import zlib

import torch

own = False

BLOCK = 32                                                      # values of a quantized block, along the head
BYTES = {"bf16": 2.0, "q8_0": 34 / BLOCK, "q4_0": 18 / BLOCK}   # a stored value
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS, THETA = 1e-6, 1e6
TILE = 32                                                       # tokens that a page holds together


def listed():
    return [
        # one decode step of a batch: normed heads, k and v into the cache; the launches are the cost
        {"name": "heads_step", "op": "heads", "heads": 16, "kv": 8, "dim": 128, "tokens": 48, "input": "bf16", "norm": True, "far": 100000, "cache": "q8_0", "page": 64},
        # a prompt's q and k before its attention
        {"name": "heads_prompt", "op": "heads", "heads": 16, "kv": 8, "dim": 128, "tokens": 4100, "input": "bf16", "norm": True, "far": 0, "cache": "", "page": 64},
        # a ragged pack straight from f32 linears, heads of 64 without groups or norms
        {"name": "heads_f32", "op": "heads", "heads": 20, "kv": 20, "dim": 64, "tokens": 7305, "input": "f32", "norm": False, "far": 0, "cache": "", "page": 64},
        # long prompts, attended and kept
        {"name": "heads_long", "op": "heads", "heads": 32, "kv": 8, "dim": 128, "tokens": 32768, "input": "bf16", "norm": True, "far": 0, "cache": "q8_0", "page": 128},
        # a batch of prompts of odd lengths starts
        {"name": "place_prompts", "op": "place", "n": 24, "longest": 1000, "beams": 1, "room": 129, "page": 64, "held": 0, "mix": 1},
        # a full batch with beams
        {"name": "place_beams", "op": "place", "n": 256, "longest": 2000, "beams": 4, "room": 256, "page": 64, "held": 0, "mix": 2},
        # sequences of all ages go on by a token each
        {"name": "place_step", "op": "place", "n": 200, "longest": 1, "beams": 1, "room": 0, "page": 64, "held": 6000, "mix": 3},
        # one request
        {"name": "select_one", "op": "select", "n": 1, "beams": 4, "vocab": 32000, "count": 4, "input": "f32", "stop": False},
        # a batch, some beams ended, an odd vocabulary in bf16, twice as many candidates as beams
        {"name": "select_bf16", "op": "select", "n": 16, "beams": 5, "vocab": 151111, "count": 10, "input": "bf16", "stop": True},
        # a full batch
        {"name": "select_full", "op": "select", "n": 64, "beams": 8, "vocab": 128000, "count": 8, "input": "f32", "stop": True},
        # a few requests' beams
        {"name": "reorder_step", "op": "reorder", "n": 8, "beams": 4, "longest": 2000, "layers": 28, "kv": 8, "dim": 128, "type": "q8_0", "page": 64, "mix": 4},
        # a full batch's, in the widest type
        {"name": "reorder_full", "op": "reorder", "n": 64, "beams": 8, "longest": 500, "layers": 28, "kv": 8, "dim": 128, "type": "bf16", "page": 64, "mix": 5},
    ]


def _between(rng, lo, hi):
    """A whole number, spread over its logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["heads", "heads", "place", "select", "select", "reorder"])
    if op == "heads":
        heads, kv = rng.choice([(12, 12), (16, 8), (32, 8), (20, 20), (8, 1), (28, 4), (16, 2), (40, 8)])
        c = {"op": op, "heads": heads, "kv": kv, "dim": rng.choice([64, 128, 128]), "input": rng.choice(["bf16", "bf16", "f32"]),
             "norm": rng.random() < 0.7, "far": rng.choice([0, 5000, 1000000]), "cache": rng.choice(["", "bf16", "q8_0"]), "page": rng.choice([32, 64, 96, 128])}
        return {**c, "tokens": _between(rng, 1, min(32768, 500000 // (heads + 2 * kv)))}
    if op == "place":
        c = {"op": op, "n": _between(rng, 1, 500), "beams": rng.choice([1, 1, 2, 3, 4, 8]), "page": rng.choice([32, 64, 96, 128, 256]), "mix": rng.randrange(0, 1000)}
        if rng.random() < 0.3:
            return {**c, "beams": 1, "room": 0, "longest": _between(rng, 1, 40), "held": _between(rng, 1, 30000)}
        return {**c, "room": _between(rng, 1, 500), "longest": _between(rng, 1, 200000 // c["n"]), "held": 0}
    if op == "select":
        n, beams = _between(rng, 1, 64), rng.choice([1, 2, 3, 4, 5, 8, 12])
        c = {"op": op, "n": n, "beams": beams, "vocab": _between(rng, 1000, min(200000, 60000000 // (n * beams)))}
        return {**c, "count": rng.choice([beams, 2 * beams, 1, 16]), "input": rng.choice(["f32", "f32", "bf16"]), "stop": rng.random() < 0.5}
    n, beams = _between(rng, 1, 64), rng.choice([2, 3, 4, 5, 8])
    c = {"op": op, "n": n, "beams": beams, "longest": _between(rng, 1, 16000 // n), "layers": rng.choice([1, 6, 24, 28, 36]),
         "type": rng.choice(["bf16", "q8_0", "q4_0"]), "page": rng.choice([32, 64, 96, 128]), "mix": rng.randrange(0, 1000)}
    kv, dim = rng.choice([(8, 128), (2, 128), (4, 64), (1, 128)])
    return {**c, "kv": kv, "dim": dim}


def _lengths(case):
    """The requests' lengths, spread up to the longest, itself among them."""
    rng, longest = random.Random(case["mix"]), case["longest"]
    return [longest] + [_between(rng, 1, longest) if k % 2 else rng.randint(1, longest) for k in range(1, case["n"])]


def _parents(case):
    """Beams' parents, as a search gives them: mostly the better beams."""
    rng, b = random.Random(case["mix"] + 1), case["beams"]
    return [[min(rng.randrange(b), rng.randrange(b)) if rng.random() < 0.5 else j for j in range(b)] for _ in range(case["n"])]


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


def _beams():
    from mold_amd import beams
    return beams


def _cache(case, kind, pages):
    from mold_amd import GgmlDType
    return _text().KvCache(pages, case["kv"], case["dim"], page_tokens=case["page"],
                           dtype={"bf16": GgmlDType.BF16, "q8_0": GgmlDType.Q8_0, "q4_0": GgmlDType.Q4_0}[kind], device="cuda")


# ------------------------------------------------------------------ inputs

def prepare(case, seed):
    return {"heads": _prepare_heads, "place": _prepare_place, "select": _prepare_select, "reorder": _prepare_reorder}[case["op"]](case, seed)


def _heads_inputs(case, seed):
    t, h, kv, d = case["tokens"], case["heads"], case["kv"], case["dim"]
    qkv = _rows(seed, "qkv", t, h + 2 * kv, d, dtype=DTYPES[case["input"]])       # one projection's output, its parts side by side
    g = _gen(seed, "positions")
    if case["far"]:
        pos = torch.randint(0, case["far"], (t,), device="cuda", generator=g)
    else:                                                        # packed prompts: each starts anew
        start = torch.rand(t, device="cuda", generator=g) < 1 / 700
        at = torch.arange(t, device="cuda")
        pos = at - torch.cummax(torch.where(start, at, 0), 0).values
    half = d // 2
    freq = THETA ** (-torch.arange(half, device="cuda", dtype=torch.float32) / half)
    qw, kw = (1 + 0.1 * torch.randn((2, d), device="cuda", generator=g)).unbind() if case["norm"] else (None, None)
    return qkv[:, :h], qkv[:, h:h + kv], qkv[:, h + kv:], pos, freq, qw, kw


def _slots(case, seed):
    """Pages of the pool in no order, and the tokens' slots in them, one after another."""
    page, t = case["page"], torch.arange(case["tokens"], device="cuda")
    used = -(-case["tokens"] // page)
    order = torch.randperm(used + 3, device="cuda", generator=_gen(seed, "pages"))[:used]
    return used + 3, order[t // page] * page + t % page


def _prepare_heads(case, seed):
    state = {"op": "heads", "kind": case["cache"], "dtype": case["input"]}
    state["in"] = _heads_inputs(case, seed)
    if case["cache"]:
        pool, state["slots"] = _slots(case, seed)
        state["cache"] = _cache(case, case["cache"], pool) if own else _plain_pool(case["cache"], pool * case["page"], case["kv"], case["dim"])
    return state


def _place_sizes(case):
    """Counts, what is held, the table's width and the pages that the cache has."""
    counts, page = _lengths(case), case["page"]
    rng = random.Random(case["mix"] + 2)
    held = [rng.randint(0, case["held"]) for _ in counts]
    width = max(-(-(c + h + case["room"]) // page) for c, h in zip(counts, held)) + 1
    need = [_need(c + h, case, page) for c, h in zip(counts, held)]
    return counts, held, width, sum(s + case["beams"] * (w - s) for s, w in need) + 5


def _need(length, case, page):
    """A request's pages that all its beams share, and a beam's pages."""
    return (length // page if case["beams"] > 1 else 0), -(-(length + case["room"]) // page)


def _prepare_place(case, seed):
    counts, held, width, pool = _place_sizes(case)
    dev = dict(dtype=torch.int32, device="cuda")
    state = {"op": "place", "counts": torch.tensor(counts, **dev), "tokens": sum(counts), "width": width, "room": case["room"], "beams": case["beams"],
             "page": case["page"], "pool": pool, "held": None, "pages": torch.randperm(pool, device="cuda", generator=_gen(seed, "pages")).to(torch.int32)}
    if case["held"]:
        state["held"] = torch.tensor(held, **dev)
        per = torch.tensor([-(-(c + h) // case["page"]) for c, h in zip(counts, held)], device="cuda")
        first = torch.cumsum(per, 0) - per
        column = torch.arange(width, device="cuda")
        at = first[:, None] + column
        state["table"] = torch.where(column < per[:, None], state["pages"][at.clamp(max=pool - 1)], -1).to(torch.int32)
    if own:
        state["cache"] = _cache({"kv": 1, "dim": 64, "page": case["page"]}, "q4_0", pool)
    return state


def _select_inputs(case, seed):
    n, b, v = case["n"], case["beams"], case["vocab"]
    g = _gen(seed, "logits")
    x = torch.randn((n, b, v), device="cuda", generator=g).mul_(1.5 + 2 * torch.rand((n, b, 1), device="cuda", generator=g))
    scores = -10 * torch.rand((n, b), device="cuda", generator=g)
    last, stop = None, None
    if case["stop"]:
        stop = 2
        last = torch.where(torch.rand((n, b), device="cuda", generator=g) < 0.2, stop, 7 + torch.arange(b, device="cuda"))
    return x.to(DTYPES[case["input"]]), scores, last, stop


def _prepare_select(case, seed):
    logits, scores, last, stop = _select_inputs(case, seed)
    return {"op": "select", "logits": logits, "scores": scores, "last": last, "stop": stop, "count": case["count"]}


def _prepare_reorder(case, seed):
    n, b, page, kv, dim, kind = (case[k] for k in ("n", "beams", "page", "kv", "dim", "type"))
    lengths = torch.tensor(_lengths(case), device="cuda")
    full, width = lengths // page, case["longest"] // page + 2
    need = full + b * 2                                          # shared pages, then the last two of each beam
    pool = int(need.sum())
    order = torch.randperm(pool, device="cuda", generator=_gen(seed, "pages"))
    first = (torch.cumsum(need, 0) - need)[:, None, None]
    column, beam = torch.arange(width, device="cuda"), torch.arange(b, device="cuda")[:, None]
    own_at = full[:, None, None] + 2 * beam + (column - full[:, None, None])
    at = first + torch.where(column < full[:, None, None], column, own_at)
    held = column < full[:, None, None] + 2
    table = torch.where(held, order[at.clamp(max=pool - 1)], -1).to(torch.int32).reshape(n * b, width).contiguous()
    size = int(2 * kv * dim * page * BYTES[kind])
    state = {"op": "reorder", "table": table, "lengths": lengths.to(torch.int32).repeat_interleave(b), "page": page, "heads": kv, "pool": pool,
             "parents": torch.tensor(_parents(case), dtype=torch.int32, device="cuda"), "pools": [], "caches": []}
    for layer in range(case["layers"]):
        x = torch.randint(0, 256, (pool * size,), dtype=torch.uint8, device="cuda", generator=_gen(seed, f"pool{layer}"))
        if own:
            state["caches"].append(_cache(case, kind, pool))
            state["caches"][-1].data.copy_(x)
        else:
            state["pools"].append(x)
    if own:
        state["states"] = _beams().BeamStates(state["caches"])
    return state


# ------------------------------------------------------------------ plain forms

def _plain_pool(kind, slots, kv, d):
    """A cache as plain tensors, keys first: values, or whole numbers and the scale of each block."""
    if kind == "bf16":
        return {"x": torch.zeros((2, slots, kv, d), dtype=torch.bfloat16, device="cuda")}
    return {"x": torch.zeros((2, slots, kv, d), dtype=torch.int8, device="cuda"),
            "d": torch.zeros((2, slots, kv, d // BLOCK), dtype=torch.float16, device="cuda")}


def _plain_rotated(x, weight, angle):
    """bf16 of x [tokens, heads, dim] normed (with a weight) and rotated by angle [tokens, dim / 2]."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight
    a, b = x.chunk(2, -1)
    c, s = angle.cos().float()[:, None], angle.sin().float()[:, None]
    return torch.cat([a * c - b * s, b * c + a * s], -1).bfloat16()


def _plain_heads(s):
    q, k, v, pos, freq, qw, kw = s["in"]
    angle = pos.double()[:, None] * freq.double()                # far positions: f32 has no fraction of a turn left
    q, k = _plain_rotated(q, qw, angle), _plain_rotated(k, kw, angle)
    if not s["kind"]:
        return q, k
    pool, slots, kv = s["cache"], s["slots"], torch.stack([k.float(), v.float()])
    if s["kind"] == "bf16":
        pool["x"][:, slots] = kv.bfloat16()
        got = pool["x"][:, slots]
    else:
        b = kv.unflatten(-1, (-1, BLOCK))
        d = b.abs().amax(-1, keepdim=True) / 127.0
        y = b * torch.where(d != 0, 1.0 / d, torch.zeros_like(d))
        y = torch.where(y.abs() < 0.5, torch.zeros_like(y), torch.trunc(y + torch.copysign(torch.full_like(y, 0.5), y)))   # halves away from zero
        pool["x"][:, slots] = y.flatten(-2).to(torch.int8)
        pool["d"][:, slots] = d.squeeze(-1).half()
        got = (pool["x"][:, slots].float().unflatten(-1, (-1, BLOCK)) * pool["d"][:, slots].float().unsqueeze(-1)).flatten(-2).bfloat16()
    return q, k, got[0], got[1]


def _plain_place(s):
    counts, page, n, tokens = s["counts"].long(), s["page"], s["counts"].shape[0], s["tokens"]
    ends = torch.cumsum(counts, 0)
    seq = torch.repeat_interleave(torch.arange(n, device="cuda"), counts, output_size=tokens)
    pos = torch.arange(tokens, device="cuda") - (ends - counts)[seq]
    if s["held"] is not None:
        pos = pos + s["held"].long()[seq]
        return s["table"].long()[seq, pos // page] * page + pos % page, pos, (s["held"].long() + counts).int()
    beams, width = s["beams"], s["width"]
    shared = counts // page if beams > 1 else torch.zeros_like(counts)
    columns = -(-(counts + s["room"]) // page)
    need = shared + beams * (columns - shared)
    first = torch.cumsum(need, 0) - need
    column, beam = torch.arange(width, device="cuda"), torch.arange(beams, device="cuda")[:, None]
    sh, co = shared[:, None, None], columns[:, None, None]
    at = first[:, None, None] + torch.where(column < sh, column, sh + beam * (co - sh) + column - sh)
    table = torch.where(column < co, s["pages"][at.clamp(max=s["pool"] - 1)], -1)
    slots = table[:, 0].long()[seq, pos // page] * page + pos % page
    return table.reshape(n * beams, width).int(), slots, pos, s["counts"].repeat_interleave(beams), ends - 1


def _plain_select(s):
    x, b = s["logits"].double(), s["logits"].shape[1]            # in 64 bits: beams compare by sums that lie close
    n, _, v = x.shape
    x = x - x.amax(-1, keepdim=True)
    total = x.sub_(x.exp().sum(-1, keepdim=True).log()).add_(s["scores"].double()[..., None])
    if s["stop"] is not None:
        done = (s["last"] == s["stop"])[..., None]
        at_stop = torch.arange(v, device="cuda") == s["stop"]
        total = torch.where(done, torch.where(at_stop, s["scores"].double()[..., None], -math.inf), total)
    value, at = torch.sort(total.reshape(n, b * v), dim=-1, descending=True, stable=True)     # ties: the lowest beam and token first
    value, at = value[:, :s["count"]], at[:, :s["count"]]
    none = value == -math.inf
    return value.float(), torch.where(none, 0, at // v).int(), torch.where(none, -1, at % v)


def _plain_reorder(s):
    page, table, p = s["page"], s["table"], s["parents"].long()
    n, b = p.shape
    width = table.shape[1]
    beam = torch.arange(b, device="cuda")
    length = s["lengths"].view(n, b)[:, 0].long()
    full, tail = length // page, length % page
    child = p[:, None, :] == beam[:, None]                       # [n, parent, child]
    first = torch.where(child, beam, b).amin(-1)
    keeper = torch.where(child.diagonal(dim1=1, dim2=2), beam, first)       # the child that takes its parent's page on
    keeps = torch.gather(keeper, 1, p) == beam
    dead = torch.sort(torch.where(child.any(-1), b, beam), dim=-1).values
    rank = torch.cumsum((~keeps).long(), -1) - 1
    taken = torch.where(keeps, p, torch.gather(dead, 1, rank.clamp(min=0)).clamp(max=b - 1))    # whose page each beam has now
    rows = table.view(n, b, width)
    last = torch.gather(rows, 2, full[:, None, None].expand(n, b, 1)).squeeze(-1).long()
    source, target = torch.gather(last, 1, p), torch.gather(last, 1, taken)
    tiles = page // TILE
    copied = torch.arange(tiles, device="cuda") < ((tail + TILE - 1) // TILE)[:, None, None]     # [n, 1, tiles]
    copied = (copied & ~keeps[:, :, None]).reshape(n * b, 1, tiles, 1)
    source, target = torch.where(tail[:, None] > 0, source, last).reshape(-1), torch.where(tail[:, None] > 0, target, last).reshape(-1)
    for pool in s["pools"]:
        x = pool.view(-1, s["heads"], tiles, pool.numel() // (s["pool"] * s["heads"] * tiles))
        x[target] = torch.where(copied, x[source], x[target])
    column = torch.arange(width, device="cuda")
    new = torch.where(column < full[:, None, None], torch.gather(rows, 1, p[..., None].expand(n, b, width)), rows)
    here = (column == full[:, None, None]) & (tail[:, None, None] > 0)
    table.copy_(torch.where(here, target.view(n, b, 1).int(), new).reshape(n * b, width))
    return (table, *s["pools"])


def run(state):
    op = state["op"]
    if not own:
        return {"heads": _plain_heads, "place": _plain_place, "select": _plain_select, "reorder": _plain_reorder}[op](state)
    if op == "heads":
        q, k, v, pos, freq, qw, kw = state["in"]
        if not state["kind"]:
            return _text().rotate_heads(q, k, pos, freq, q_weight=qw, k_weight=kw, eps=EPS)
        q, k = state["cache"].append_rotated(q, k, v, state["slots"], pos, freq, q_weight=qw, k_weight=kw, eps=EPS, keys=True)
        return (q, k, *state["cache"].read(state["slots"], dtype=torch.bfloat16))
    if op == "place":
        if state["held"] is not None:
            return state["cache"].extend(state["table"], state["held"], counts=state["counts"], tokens=state["tokens"])
        return state["cache"].place(state["counts"], state["tokens"], state["width"], room=state["room"], beams=state["beams"], pages=state["pages"])
    if op == "select":
        return _beams().select_beams(state["logits"], state["scores"], count=state["count"], last=state["last"], stop=state["stop"])
    state["states"].reorder(state["table"], state["lengths"], state["parents"])
    return (state["table"], *(c.data for c in state["caches"]))


# ------------------------------------------------------------------ what a pass needs

def work(case):
    op = case["op"]
    if op == "heads":
        t, h, kv, d = (case[k] for k in ("tokens", "heads", "kv", "dim"))
        size = 4 if case["input"] == "f32" else 2
        moved = t * d * (h + kv) * (size + 2)
        if case["cache"]:
            moved += t * d * kv * (size + 2 * (2 * BYTES[case["cache"]] + 2)) + 16 * t      # v; both stored, read back and given; slots twice
        return {"bytes": moved + 8 * t, "flops": 10 * t * d * (h + kv)}
    if op == "place":
        counts, held, width, _ = _place_sizes(case)
        need = [_need(c, case, case["page"])[1] for c in counts]
        rows = case["n"] * case["beams"] * width if not case["held"] else sum(-(-c // case["page"]) + 1 for c in counts)
        return {"bytes": 16 * sum(counts) + 4 * rows + 4 * sum(need) + 12 * case["n"], "flops": 4 * sum(counts)}
    if op == "select":
        rows = case["n"] * case["beams"]
        return {"bytes": rows * (case["vocab"] * (4 if case["input"] == "f32" else 2) + 12) + 16 * case["n"] * case["count"], "flops": 4 * rows * case["vocab"]}
    page, tokens = case["page"], 0
    for length, parents in zip(_lengths(case), _parents(case)):
        tokens += (length % page) * (case["beams"] - len(set(parents)))
    rows = case["n"] * case["beams"]
    moved = case["layers"] * 2 * tokens * 2 * case["kv"] * case["dim"] * BYTES[case["type"]]
    return {"bytes": moved + 8 * rows * (case["longest"] // page + 1) + 8 * rows, "flops": rows}


# ------------------------------------------------------------------ 64 bits

def _exact_rotated(x, weight, turn):
    x = x.double()
    if weight is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * weight.double()
    half = x.shape[-1] // 2
    z = torch.complex(x[..., :half], x[..., half:]) * turn[:, None]
    return torch.cat([z.real, z.imag], -1)


def _exact_stored(kind, x):
    """The values that x's stored form stands for, by the definition; x as the cache takes it, in bf16."""
    x = x.bfloat16().double()
    if kind == "bf16":
        return x
    b = x.reshape(-1, BLOCK)
    d = b.abs().max(1, keepdim=True).values / 127
    q = torch.where(d > 0, (b.abs() / d.clamp(min=1e-300) + 0.5).floor() * b.sign(), torch.zeros_like(b))
    return (q * d.half().double()).reshape(x.shape)


def _exact_heads(case, seed):
    q, k, v, pos, freq, qw, kw = _heads_inputs(case, seed)
    angle = pos.double()[:, None] * freq.double()
    turn = torch.polar(torch.ones_like(angle), angle)
    q, k = _exact_rotated(q, qw, turn), _exact_rotated(k, kw, turn)
    if not case["cache"]:
        return q, k
    return q, k, _exact_stored(case["cache"], k), _exact_stored(case["cache"], v)


def _exact_select(case, seed):
    logits, scores, last, stop = _select_inputs(case, seed)
    n, b, v = logits.shape
    k = case["count"]
    out = (torch.full((n, k), -math.inf, dtype=torch.float64), torch.zeros((n, k), dtype=torch.int32), torch.full((n, k), -1))
    for i in range(n):
        found = []
        for j in range(b):
            score = float(scores[i, j])
            if stop is not None and int(last[i, j]) == stop:
                found.append((score, j, stop))
                continue
            x = logits[i, j].double()
            total = score + torch.log_softmax(x, 0)
            least = torch.topk(x, min(k, v)).values[-1]
            at = torch.nonzero(x >= least).flatten()
            found += [(t, j, a) for t, a in zip(total[at].tolist(), at.tolist())]
        found.sort(key=lambda f: (-f[0], f[1], f[2]))
        for m, (t, j, a) in enumerate(found[:k]):
            out[0][i, m], out[1][i, m], out[2][i, m] = t, j, a
    return out


def exact(case, seed):
    if case["op"] == "heads":
        return _exact_heads(case, seed)
    if case["op"] == "select":
        return _exact_select(case, seed)
    return None                                                  # whole numbers and bytes that are moved
