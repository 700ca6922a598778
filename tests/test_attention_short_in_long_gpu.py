"""Rows that see few keys in calls that have room for more: the 16-bit kernels
hold their P and dS as two terms whatever the extents of the tensors (bounds of
attention_reference.py with the square of the unit roundoff)."""
import pytest
import torch

import bloth_b200
from attention_reference import U, attention, check, sequences

pytestmark = pytest.mark.gpu

BF, FH = torch.bfloat16, torch.float16


def _run(dev, dtype, D, B, Sq, Sk, causal=True, window=None, q_lens=None, k_lens=None, cu=None,
         cu_k=None, seed=0, names=("o", "dq", "dk", "dv"), rows=slice(None)):
    gen = torch.Generator(device=dev).manual_seed(seed)
    rand = lambda s, h: torch.randn(B, s, h, D, generator=gen, device=dev).to(dtype)  # noqa: E731
    q, do, k, v = rand(Sq, 4), rand(Sq, 4), rand(Sk, 2), rand(Sk, 2)
    want = attention(q, k, v, do, sequences(B, Sq, Sk, q_lens, k_lens, cu, cu_k), causal, window,
                     inner=U[dtype] ** 2)
    t = lambda x: x and torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    q, k, v = (x.requires_grad_(True) for x in (q, k, v))
    o = bloth_b200.fused_attention(q, k, v, causal=causal, window=window, q_lens=t(q_lens),
                                   k_lens=t(k_lens), cu_seqlens=t(cu), cu_seqlens_k=t(cu_k))
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(o, (q, k, v), do)), o=o.detach())
    assert bloth_b200.device_fault() == 0
    for n in names:
        val, err = want[n]
        check(got[n][:, rows], (val[:, rows], err[:, rows]), n)


@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_short_documents(cuda, dtype, D, causal):
    cu = [0, 2, 5, 22, 24, 89, 217, 217, 218, 345, 349]
    _run(cuda, dtype, D, 1, 349, 349, causal, cu=cu)


@pytest.mark.parametrize("dtype", [BF, FH])
def test_packed_short_documents_with_their_own_keys(cuda, dtype):
    _run(cuda, dtype, 128, 1, 400, 190, cu=[0, 10, 300, 400], cu_k=[0, 100, 102, 190])


@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_padded_short_sequences(cuda, dtype, D, causal):
    lens = [128, 2, 3, 77, 0]
    _run(cuda, dtype, D, 5, 300, 300, causal, q_lens=lens, k_lens=lens)


@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Sq", [1, 4, 40])
def test_short_caches_in_long_ones(cuda, dtype, D, Sq):
    _run(cuda, dtype, D, 4, Sq, 700, k_lens=[128, 41, 60, 100])


@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_first_tile_of_long_sequences(cuda, dtype, D):
    # rows 0..127 see 1 to 128 keys each; dK and dV sum over longer rows as well
    _run(cuda, dtype, D, 1, 700, 700, names=("o", "dq"), rows=slice(0, 128))
