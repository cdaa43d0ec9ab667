"""The GGUF text decoder: prompt and step forwards against a float64 model of the same
(dequantized) weights, one another, and a captured step.

Bounds: a layer's activations are rounded to bf16 about eight times (norm outputs, q, k, v,
probabilities, attention, MLP input), 1.7e-3 relative on average each; two layers and the output
projection's input make 17 roundings, 7e-3 together if independent.  2e-2 is asserted, and for
the cache types their own error on top: 5e-2 for Q8_0 (7.8 bits a value), which the comparison
with a BF16 cache must show to be the cache's."""
import pytest

torch = pytest.importorskip("torch")

from mold_amd import Device, GgmlDType, QTensor
from mold_amd.text_decoder import TextConfig, TextDecoder

pytestmark = pytest.mark.gpu
CFG = TextConfig(hidden=512, heads=8, kv_heads=2, head_dim=64, layers=2, rope_theta=1e4)
VOCAB, FFN = 1000, 1024
PROMPTS = [[5, 17, 300, 42, 7], [999], list(range(100, 170)), [3, 3, 3]]


@pytest.fixture(scope="module")
def model():
    dev, g = Device(0), torch.Generator(device="cuda").manual_seed(0)
    rand = lambda *s, scale=0.04: torch.randn(s, device="cuda", generator=g) * scale
    w, dense = {}, {}

    def linear(name, n, k):
        qt = QTensor.quantize(dev, rand(n, k), GgmlDType.Q8_0)
        w[name], dense[name] = qt, qt.dequantize().double()

    def norm(name, n):
        w[name] = 1 + rand(n, scale=0.1)
        dense[name] = w[name].double()
    w["token_embd.weight"] = rand(VOCAB, CFG.hidden, scale=1.0)
    dense["token_embd.weight"] = w["token_embd.weight"].double()
    norm("output_norm.weight", CFG.hidden)
    linear("output.weight", VOCAB, CFG.hidden)
    for i in range(CFG.layers):
        b, d = f"blk.{i}", CFG.head_dim
        for name, n, k in (("attn_q", CFG.heads * d, CFG.hidden), ("attn_k", CFG.kv_heads * d, CFG.hidden), ("attn_v", CFG.kv_heads * d, CFG.hidden),
                           ("attn_output", CFG.hidden, CFG.heads * d), ("ffn_gate", FFN, CFG.hidden), ("ffn_up", FFN, CFG.hidden),
                           ("ffn_down", CFG.hidden, FFN)):
            linear(f"{b}.{name}.weight", n, k)
        for name, n in (("attn_norm", CFG.hidden), ("ffn_norm", CFG.hidden), ("attn_q_norm", d), ("attn_k_norm", d)):
            norm(f"{b}.{name}.weight", n)
    return w, dense


def _reference(dense, tokens):
    """float64 logits after every token of one prompt."""
    c, n = CFG, len(tokens)
    x = dense["token_embd.weight"][torch.tensor(tokens, device="cuda")]
    norm = lambda t, name: t * torch.rsqrt(t.square().mean(-1, keepdim=True) + c.eps) * dense[name]
    half = c.head_dim // 2
    angle = torch.arange(n, device="cuda").double()[:, None] * c.rope_theta ** (-torch.arange(half, device="cuda").double() / half)

    def rope(t):
        z = torch.complex(t[..., :half], t[..., half:]) * torch.polar(torch.ones_like(angle), angle)[:, None]
        return torch.cat([z.real, z.imag], -1)
    for i in range(c.layers):
        b = f"blk.{i}."
        h = norm(x, b + "attn_norm.weight")
        q, k, v = ((h @ dense[f"{b}attn_{s}.weight"].t()).unflatten(-1, (-1, c.head_dim)) for s in "qkv")
        q, k = rope(norm(q, b + "attn_q_norm.weight")), rope(norm(k, b + "attn_k_norm.weight"))
        k, v = (t.repeat_interleave(c.heads // c.kv_heads, 1).transpose(0, 1) for t in (k, v))
        s = q.transpose(0, 1) @ k.transpose(1, 2).contiguous() / c.head_dim ** 0.5
        s = s + torch.full_like(s, float("-inf")).triu(1)
        a = (torch.softmax(s, -1) @ v.contiguous()).transpose(0, 1).flatten(1)
        x = x + a @ dense[b + "attn_output.weight"].t()
        h = norm(x, b + "ffn_norm.weight")
        g = torch.nn.functional.silu(h @ dense[b + "ffn_gate.weight"].t()) * (h @ dense[b + "ffn_up.weight"].t())
        x = x + g @ dense[b + "ffn_down.weight"].t()
    return norm(x, "output_norm.weight") @ dense["output.weight"].t()


def _err(a, b):
    return ((a.double() - b).norm() / b.norm()).item()


def _decoder(model, dtype, pages=40):
    return TextDecoder(CFG, model[0], pages=pages, page_tokens=32, cache_dtype=dtype)


@pytest.mark.parametrize("dtype,bound", [(GgmlDType.BF16, 2e-2), (GgmlDType.Q8_0, 5e-2)], ids=lambda x: getattr(x, "name", ""))
def test_prompts_then_steps(model, dtype, bound):
    """Each prompt as if alone, then 40 given tokens of each, past a page's end."""
    dec = _decoder(model, dtype)
    logits = dec.prefill(PROMPTS, room=40)
    more = torch.randint(0, VOCAB, (40, len(PROMPTS)), generator=torch.Generator().manual_seed(3))
    refs = [_reference(model[1], p + more[:, i].tolist()) for i, p in enumerate(PROMPTS)]
    for i, p in enumerate(PROMPTS):
        assert _err(logits[i], refs[i][len(p) - 1]) < 2e-2, i
    for t in range(40):
        logits = dec.step(more[t].cuda())
        for i, p in enumerate(PROMPTS):
            assert _err(logits[i], refs[i][len(p) + t]) < bound, (t, i)
    assert dec.lengths.tolist() == [len(p) + 40 for p in PROMPTS]


def test_captured_step(model):
    """A step replayed from a graph gives what the eager one gives, token after token."""
    eager, graphed = _decoder(model, GgmlDType.Q8_0), _decoder(model, GgmlDType.Q8_0)
    first = eager.prefill(PROMPTS, room=20).argmax(-1)
    graphed.prefill(PROMPTS, room=20)
    token = first.clone()
    start = graphed.lengths.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        graphed.step(token)                                  # workspaces of this stream
        graphed.lengths.copy_(start)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            logits = graphed.step(token)
    torch.cuda.current_stream().wait_stream(s)
    graphed.lengths.copy_(start)
    for t in range(20):
        want = eager.step(token)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(logits, want), t
        token.copy_(want.argmax(-1))


def test_generate_and_refusals(model):
    dec = _decoder(model, GgmlDType.BF16)
    out = dec.generate(PROMPTS, 6)
    assert out.shape == (4, 6)
    assert torch.equal(out, dec.generate(PROMPTS, 6))
    stopped = dec.generate(PROMPTS, 6, stop=int(out[0, 0]))
    assert (stopped[0] == out[0, 0]).all()
    for prompts in ([], [[]], [[1], []]):
        with pytest.raises(ValueError):
            dec.prefill(prompts)
    with pytest.raises(ValueError):
        dec.prefill([[1] * 64] * 30)
    fresh = _decoder(model, GgmlDType.BF16, pages=2)
    with pytest.raises(ValueError):
        fresh.step(torch.zeros(1, dtype=torch.int64, device="cuda"))
    fresh.prefill([[1] * 31, [2, 3]])                          # a page each, one token left in the first
    for t in range(3):
        logits = fresh.step(torch.tensor([4, 5], device="cuda"))
        assert torch.isfinite(logits[1]).all() and bool(torch.isfinite(logits[0]).all()) == (t == 0)
