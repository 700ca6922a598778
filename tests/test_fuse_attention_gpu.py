"""HuggingFace models under flash attention, patched with fuse_attention=True,
against the same models unpatched. HuggingFace's flash attention is replaced by
a plain one with its rules: offsets if they are given, else, for one row,
documents where the positions do not go on by one."""
import sys

import pytest
import torch

import bloth_b200
from bloth_b200 import attention as binding

pytestmark = pytest.mark.gpu


def _plain_flash(module, q, k, v, mask, scaling=None, position_ids=None, cu_seq_lens_q=None, **kw):
    assert mask is None
    B, H, S, _ = q.shape
    k, v = (x.repeat_interleave(H // x.shape[1], 1) for x in (k, v))
    doc = torch.zeros(B, S, dtype=torch.long, device=q.device)
    if cu_seq_lens_q is not None:
        assert B == 1
        doc[0] = torch.bucketize(torch.arange(S, device=q.device), cu_seq_lens_q[1:], right=True)
    elif B == 1 and position_ids is not None:
        doc[:, 1:] = (position_ids[:, 1:] != position_ids[:, :-1] + 1).cumsum(1)
    see = (doc.unsqueeze(1) == doc.unsqueeze(2)).tril().unsqueeze(1)
    p = torch.softmax((q @ k.transpose(2, 3) * scaling).masked_fill(~see, -float("inf")), -1)
    return (p @ v).transpose(1, 2), None


@pytest.mark.parametrize("kind", ["Llama", "Qwen3"])
@pytest.mark.parametrize("call", ["whole", "two rows", "packed positions", "offsets"])
def test_flash_attention_models_match(cuda, kind, call, monkeypatch):
    transformers = pytest.importorskip("transformers")
    cfg = dict(vocab_size=128, hidden_size=128, intermediate_size=256, num_hidden_layers=2,
               num_attention_heads=4, num_key_value_heads=2, head_dim=64,
               attn_implementation="sdpa")
    models = []
    for _ in range(2):
        torch.manual_seed(0)
        models.append(getattr(transformers, kind + "ForCausalLM")(
            getattr(transformers, kind + "Config")(**cfg)).to(cuda))
        models[-1].config._attn_implementation = "flash_attention_2"
    hf, ours = models
    monkeypatch.setitem(sys.modules[type(hf).__module__].ALL_ATTENTION_FUNCTIONS,
                        "flash_attention_2", _plain_flash)
    bloth_b200.patch_model(ours, verbose=False, fuse_attention=True)
    fused, real = [], binding.fused_attention
    monkeypatch.setattr(binding, "fused_attention",
                        lambda *a, **kw: fused.append(kw) or real(*a, **kw))
    ids = torch.randint(0, 128, (2 if call == "two rows" else 1, 90), device=cuda)
    kw = {}
    if call in ("packed positions", "offsets"):
        kw["position_ids"] = torch.cat([torch.arange(n, device=cuda) for n in (33, 1, 56)])[None]
    if call == "offsets":
        cu = torch.tensor([0, 33, 34, 90], dtype=torch.int32, device=cuda)
        kw.update(cu_seq_lens_q=cu, cu_seq_lens_k=cu, max_length_q=56, max_length_k=56)
    a, b = (m(ids, use_cache=False, **kw).logits for m in models)
    assert len(fused) == (0 if call == "packed positions" else 2)
    # fp32 throughout, so the two differ in rounding order only (1e-4 as the
    # other whole-model tests)
    assert float((a - b).abs().max()) < 1e-4
    g = torch.randn_like(a)
    a.backward(g)
    b.backward(g)
    for (n, p), (_, q) in zip(hf.named_parameters(), ours.named_parameters()):
        assert float((p.grad - q.grad).abs().max()) <= 1e-4 * max(1.0, float(p.grad.abs().max())), n
