"""A text decoder made from a GGUF file: metadata to configuration, every tensor as
Content.var_builder gives it (embedding and norms in any of the file's types)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from mold_amd import Device, GgmlDType, QTensor, gguf
from mold_amd.text_decoder import TextConfig, TextDecoder
from tests.test_gpu_text_decoder import CFG, PROMPTS, VOCAB, model  # noqa: F401

META = {"general.architecture": "qwen3", "qwen3.embedding_length": 512, "qwen3.attention.head_count": 8, "qwen3.attention.head_count_kv": 2,
        "qwen3.attention.key_length": 64, "qwen3.block_count": 2, "qwen3.rope.freq_base": 1e4, "qwen3.attention.layer_norm_rms_epsilon": 1e-6}


def test_configuration():
    got = TextConfig.from_metadata(META)
    assert got == CFG
    few = {k: v for k, v in META.items() if not k.endswith(("_kv", "key_length", "freq_base", "epsilon"))}
    assert TextConfig.from_metadata(few) == TextConfig(512, 8, 8, 64, 2)
    for key in ("general.architecture", "qwen3.embedding_length", "qwen3.block_count"):
        with pytest.raises((KeyError, ValueError)):
            TextConfig.from_metadata({k: v for k, v in META.items() if k != key})


@pytest.mark.gpu
@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("embedding", [GgmlDType.Q6_K, GgmlDType.Q8_0, GgmlDType.F16, GgmlDType.F32], ids=lambda t: t.name)
def test_from_a_file(model, tmp_path, embedding, tied):
    """As the decoder of the same values in float32 tensors, bit for bit; a tied output reads the
    embedding's blocks, as float32 products of its values up to the rounding of their input to bf16."""
    dev = Device(0)
    weights = {k: w for k, w in model[0].items() if not (tied and k == "output.weight")}
    weights["token_embd.weight"] = QTensor.quantize(dev, weights["token_embd.weight"], embedding)
    # a dense projection, and biases
    weights["blk.1.attn_k.weight"] = QTensor.quantize(dev, weights["blk.1.attn_k.weight"].dequantize(), GgmlDType.F16)
    weights["blk.0.attn_q.bias"] = torch.linspace(-1, 1, 512, device="cuda")
    tensors = []
    for name, w in weights.items():
        if isinstance(w, QTensor):
            tensors.append((name, w.dtype(), w.shape, w.data()))
        else:
            tensors.append((name, GgmlDType.F32, tuple(w.shape), w.cpu().numpy().view(np.uint8)))
    path = str(tmp_path / "decoder.gguf")
    gguf.write(path, tensors, metadata=META)
    content = gguf.Content.read(path)
    cfg = TextConfig.from_metadata(content.metadata)
    assert (cfg.hidden, cfg.heads, cfg.kv_heads, cfg.head_dim, cfg.layers, cfg.rope_theta) == (512, 8, 2, 64, 2, 1e4)
    cfg = CFG                                                # its eps is stored in float32
    loaded = TextDecoder(cfg, content.var_builder(dev), pages=40, page_tokens=32, cache_dtype=GgmlDType.BF16)
    content.close()
    plain = dict(weights)
    for name in ("token_embd.weight", "blk.1.attn_k.weight"):
        plain[name] = weights[name].dequantize()
    made = TextDecoder(cfg, plain, pages=40, page_tokens=32, cache_dtype=GgmlDType.BF16)
    got, want = loaded.prefill(PROMPTS, room=4), made.prefill(PROMPTS, room=4)
    for _ in range(4):
        assert got.shape == (len(PROMPTS), VOCAB)
        if tied and embedding.is_quantized:
            # x rounded to bf16 (2^-9 / sqrt(3) of itself) and the blocks' products by bf16 dequantized values at worst (twice that)
            assert ((got - want).norm() / want.norm()).item() < 3.0 * 2.0 ** -9
        else:
            assert torch.equal(got, want)
        token = want.argmax(-1)
        got, want = loaded.step(token), made.step(token)
