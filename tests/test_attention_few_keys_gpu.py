"""Rows that see few keys: the 16-bit kernels hold P and dS as two terms there
(bounds of attention_reference.py with the square of the unit roundoff), and a
row of one key passes no gradient to q and k at all."""
import pytest
import torch

import bloth_b200
from attention_reference import U, attention, check, sequences

pytestmark = pytest.mark.gpu

BF, FH, F32 = torch.bfloat16, torch.float16, torch.float32


def _run(dev, dtype, D, B, Sq, Sk, Hq, Hk, causal=True, window=None, k_lens=None, cu=None, seed=0,
         inner=True):
    gen = torch.Generator(device=dev).manual_seed(seed)
    rand = lambda s, h: torch.randn(B, s, h, D, generator=gen, device=dev).to(dtype)  # noqa: E731
    q, do, k, v = rand(Sq, Hq), rand(Sq, Hq), rand(Sk, Hk), rand(Sk, Hk)
    want = attention(q, k, v, do, sequences(B, Sq, Sk, None, k_lens, cu), causal, window,
                     inner=U[dtype] ** 2 if inner else None)
    t = lambda x: x and torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    q, k, v = (x.requires_grad_(True) for x in (q, k, v))
    o = bloth_b200.fused_attention(q, k, v, causal=causal, window=window, k_lens=t(k_lens),
                                   cu_seqlens=t(cu))
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(o, (q, k, v), do)), o=o.detach())
    torch.cuda.synchronize()
    assert bloth_b200.device_fault() == 0
    for n, x in got.items():
        check(x, want[n], n)
    return got


@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("S", [2, 3, 17, 65, 128])
def test_short_sequences(cuda, dtype, D, S):
    _run(cuda, dtype, D, 3, S, S, 4, 2, causal=S != 17, seed=S)


@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("window", [2, 64, 128])
def test_narrow_windows(cuda, dtype, D, window):
    _run(cuda, dtype, D, 2, 391, 391, 4, 2, window=window, seed=window)


@pytest.mark.parametrize("dtype", [BF, FH])
def test_few_keys_for_many_queries(cuda, dtype):
    _run(cuda, dtype, 128, 2, 515, 100, 4, 2, causal=False, k_lens=[100, 37])
    _run(cuda, dtype, 64, 2, 4, 120, 8, 1, k_lens=[120, 9])


@pytest.mark.parametrize("dtype", [BF, FH, F32])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("case", ["token", "window", "documents", "one key"])
def test_rows_of_one_key(cuda, dtype, D, case):
    inner = dtype != F32
    if case == "token":
        got = _run(cuda, dtype, D, 3, 1, 1, 4, 2, inner=inner)
        rows = slice(None)
    elif case == "window":
        got = _run(cuda, dtype, D, 1, 321, 321, 4, 2, window=1, inner=inner)
        rows = slice(None)
    elif case == "documents":  # each document's first row
        cu = [0, 5, 6, 70, 250]
        got = _run(cuda, dtype, D, 1, 250, 250, 4, 2, cu=cu, inner=False)
        rows = cu[:-1]
    else:
        got = _run(cuda, dtype, D, 2, 200, 150, 4, 2, causal=False, k_lens=[1, 1], inner=False)
        rows = slice(None)
    assert not got["dq"][:, rows].any()
    if case != "documents":
        assert not got["dk"].any()
