"""The attention operators where users meet them: HuggingFace models patched
with fuse_attention=True against the same models unpatched, and the example
block."""
import importlib.util
import os

import pytest
import torch

import bloth_b200
from bloth_b200 import attention as binding

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _model(kind, dtype, **kw):
    transformers = pytest.importorskip("transformers")
    cfg = dict(vocab_size=128, hidden_size=128, intermediate_size=256, num_hidden_layers=2,
               num_attention_heads=4, num_key_value_heads=2, head_dim=64,
               max_position_embeddings=512, attn_implementation="sdpa")
    cfg.update(kw)
    torch.manual_seed(0)
    return getattr(transformers, kind + "ForCausalLM")(
        getattr(transformers, kind + "Config")(**cfg)).to("cuda", dtype)


@pytest.fixture
def calls(monkeypatch):
    """Calls of fused_attention made through the binding."""
    seen = []
    real = binding.fused_attention

    def spy(*a, **kw):
        seen.append(kw)
        return real(*a, **kw)

    monkeypatch.setattr(binding, "fused_attention", spy)
    return seen


@pytest.mark.parametrize("kind", ["Llama", "Qwen3", "Mistral", "Qwen2"])
def test_models_match(cuda, kind, calls):
    # fp32 throughout, so the two differ in rounding order only (1e-4 as the
    # other whole-model tests)
    hf, ours = (_model(kind, torch.float32) for _ in range(2))
    bloth_b200.patch_model(ours, verbose=False, fuse_attention=True)
    ids = torch.randint(0, 128, (2, 70), device=cuda)
    a, b = (m(ids, labels=ids, use_cache=False) for m in (hf, ours))
    assert len(calls) == 2
    assert float((a.logits - b.logits).abs().max()) < 1e-4
    a.loss.backward()
    b.loss.backward()
    for (n, p), (_, q) in zip(hf.named_parameters(), ours.named_parameters()):
        assert float((p.grad - q.grad).abs().max()) <= 1e-4 * max(1.0, float(p.grad.abs().max())), n


@pytest.mark.parametrize("kind", ["Llama", "Qwen3"])
def test_generation_matches(cuda, kind, calls):
    hf, ours = (_model(kind, torch.float32).eval() for _ in range(2))
    bloth_b200.patch_model(ours, verbose=False, fuse_attention=True)
    ids = torch.randint(0, 128, (2, 9), device=cuda)
    kw = dict(max_new_tokens=12, do_sample=False, pad_token_id=0)
    assert torch.equal(hf.generate(ids, **kw), ours.generate(ids, **kw))
    assert len(calls) == 2 * 12  # the prompt and eleven single tokens, two layers


def test_padded_batches_keep_hf_attention(cuda, calls):
    hf, ours = (_model("Llama", torch.float32).eval() for _ in range(2))
    bloth_b200.patch_model(ours, verbose=False, fuse_attention=True)
    ids = torch.randint(0, 128, (2, 20), device=cuda)
    mask = torch.ones_like(ids)
    mask[0, :6] = 0
    with torch.no_grad():
        a, b = (m(ids, attention_mask=mask).logits for m in (hf, ours))
    assert not calls
    keep = mask.bool()
    assert float((a - b)[keep].abs().max()) < 1e-4


def test_dropout_keeps_hf_attention(cuda, calls):
    ours = _model("Llama", torch.float32, attention_dropout=0.1).train()
    bloth_b200.patch_model(ours, verbose=False, fuse_attention=True)
    ours(torch.randint(0, 128, (1, 10), device=cuda))
    assert not calls


def test_sliding_window_model(cuda, calls):
    kw = dict(sliding_window=16)
    hf, ours = (_model("Mistral", torch.float32, **kw).eval() for _ in range(2))
    bloth_b200.patch_model(ours, verbose=False, fuse_attention=True)
    for n in (12, 60):
        ids = torch.randint(0, 128, (1, n), device=cuda)
        with torch.no_grad():
            a, b = (m(ids).logits for m in (hf, ours))
        assert float((a - b).abs().max()) < 1e-4


def test_without_the_flag_attention_is_hf(cuda, calls):
    ours = _model("Llama", torch.float32)
    bloth_b200.patch_model(ours, verbose=False, patch_attention=True)
    ours(torch.randint(0, 128, (1, 10), device=cuda))
    assert not calls


@pytest.mark.parametrize("dtype,bound", [(torch.bfloat16, 12 * 2.0 ** -8),
                                         (torch.float32, 1e-4)])
@pytest.mark.parametrize("tokens", [2, 67, 512])
def test_example_block(cuda, dtype, bound, tokens):
    spec = importlib.util.spec_from_file_location(
        "attention_block", os.path.join(ROOT, "examples", "attention_block.py"))
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    off = ex.run(tokens, dtype)
    assert max(off.values()) <= bound, off
