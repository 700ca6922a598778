"""Which attention calls of a patched HuggingFace model go to fused_attention
and which stay with HuggingFace, on the CPU: the rotation, fused_attention and
HuggingFace's own attention are replaced by recorders, and the rotated tensors
say that they are on a GPU."""
import sys

import pytest
import torch

import bloth_b200
from bloth_b200 import attention as binding

transformers = pytest.importorskip("transformers")

LAYERS = 2


class OnGpu(torch.Tensor):
    is_cuda = property(lambda self: True)


@pytest.fixture
def model(monkeypatch):
    """model(implementation): a patched model, with .core and .hf, the keyword
    arguments of the calls that went either way."""
    def make(name, kind="Llama", **kw):
        cfg = dict(vocab_size=64, hidden_size=128, intermediate_size=256, head_dim=64,
                   num_hidden_layers=LAYERS, num_attention_heads=2, num_key_value_heads=1,
                   attn_implementation="sdpa")
        m = getattr(transformers, kind + "ForCausalLM")(
            getattr(transformers, kind + "Config")(**cfg, **kw)).eval()
        bloth_b200.patch_model(m, patch_norms=False, verbose=False, fuse_attention=True)
        m.core, m.hf = [], []

        def core(q, k, v, **kw):
            m.core.append(kw)
            return torch.zeros(q.shape)

        def own(module, q, k, v, mask, **kw):
            m.hf.append(kw)
            return torch.zeros(q.transpose(1, 2).shape), None

        monkeypatch.setattr(binding, "fused_attention", core)
        monkeypatch.setattr(binding, "apply_rope_qk", lambda q, k, **kw: (
            q.as_subclass(OnGpu), k.as_subclass(OnGpu)))
        hf = sys.modules[type(m).__module__]
        monkeypatch.setitem(hf.ALL_ATTENTION_FUNCTIONS, name, own)
        monkeypatch.setattr(hf, "eager_attention_forward", own)
        m.config._attn_implementation = name
        return m
    return make


def _run(m, batch=1, tokens=12, **kw):
    with torch.no_grad():
        m(torch.zeros(batch, tokens, dtype=torch.long), use_cache=False, **kw)
    assert len(m.core) + len(m.hf) == LAYERS
    return len(m.core) == LAYERS


RESTART = torch.tensor([[0, 1, 2, 3, 4, 0, 1, 2, 3, 4, 5, 6]])


@pytest.mark.parametrize("name", ["sdpa", "flash_attention_2", "flash_attention_3"])
@pytest.mark.parametrize("batch", [1, 2])
def test_whole_sequences_are_fused(model, name, batch):
    assert _run(model(name), batch)


def test_packed_positions_under_flash_stay(model):
    # no mask, one row, positions that start again: HF takes them for documents
    m = model("flash_attention_2")
    assert not _run(m, position_ids=RESTART)
    assert torch.equal(m.hf[0]["position_ids"], RESTART)


def test_positions_that_go_on_are_one_sequence(model):
    assert _run(model("flash_attention_2"), position_ids=torch.arange(5, 17).unsqueeze(0))


def test_one_token_is_one_sequence(model):
    assert _run(model("flash_attention_2"), tokens=1, position_ids=torch.tensor([[37]]))


def test_packed_positions_of_several_rows_are_ignored(model):
    # HF looks at the positions of one row only
    assert _run(model("flash_attention_2"), 2, position_ids=RESTART.expand(2, 12))


def test_packed_positions_under_sdpa_have_a_mask(model):
    assert not _run(model("sdpa"), position_ids=RESTART)


@pytest.mark.parametrize("name", ["sdpa", "flash_attention_2"])
def test_offsets_are_passed_on(model, name):
    cu = torch.tensor([0, 5, 12], dtype=torch.int32)
    m = model(name)
    assert _run(m, cu_seq_lens_q=cu, cu_seq_lens_k=cu, max_length_q=7, max_length_k=7)
    assert m.core[0]["cu_seqlens"] is cu and m.core[0]["cu_seqlens_k"] is cu


def test_offsets_win_over_positions(model):
    cu = torch.tensor([0, 5, 12], dtype=torch.int32)
    m = model("flash_attention_2")
    assert _run(m, position_ids=RESTART, cu_seq_lens_q=cu, cu_seq_lens_k=cu, max_length_q=7,
                max_length_k=7)
    assert m.core[0]["cu_seqlens"] is cu


@pytest.mark.parametrize("name", ["sdpa", "flash_attention_2"])
def test_offsets_over_several_rows_stay(model, name):
    # HF flattens the rows before it applies the offsets
    cu = torch.tensor([0, 5, 12, 24], dtype=torch.int32)
    assert not _run(model(name), 2, cu_seq_lens_q=cu, cu_seq_lens_k=cu, max_length_q=12,
                    max_length_k=12)


@pytest.mark.parametrize("name", ["sdpa", "flash_attention_2"])
def test_paged_caches_stay(model, name):
    m = model(name)
    attn = m.model.layers[0].self_attn
    cos = torch.ones(1, 12, 64)
    attn(torch.zeros(1, 12, 128), (cos, cos), None, cache=object())
    assert len(m.hf) == 1 and not m.core


@pytest.mark.parametrize("name", ["eager", "paged|sdpa", "paged|flash_attention_2", "my_attention"])
def test_other_implementations_stay(model, name):
    # without a mask these are not causal, or find their keys elsewhere
    m = model(name)
    attn = m.model.layers[0].self_attn
    cos = torch.ones(1, 12, 64)
    attn(torch.zeros(1, 12, 128), (cos, cos), None)
    assert len(m.hf) == 1 and not m.core


@pytest.mark.parametrize("first", [dict(patch_attention=True), dict(fuse_attention=True)])
def test_fusing_a_model_that_is_patched_already(model, first, capsys):
    m = model("sdpa")
    for layer in m.model.layers:  # as before any patch
        del layer.self_attn._bloth_attention, layer.self_attn.__dict__["forward"]
    bloth_b200.patch_model(m, patch_norms=False, verbose=False, **first)
    fused = "fuse_attention" in first
    assert _run(m) == fused
    m.core.clear(), m.hf.clear()
    bloth_b200.patch_model(m, patch_norms=False, fuse_attention=True)
    assert (f"Patched {LAYERS} attention layer(s)" in capsys.readouterr().out) == (not fused)
    assert _run(m)
    # patch_attention alone takes nothing back
    m.core.clear(), m.hf.clear()
    bloth_b200.patch_model(m, patch_norms=False, verbose=False, patch_attention=True)
    assert _run(m)
