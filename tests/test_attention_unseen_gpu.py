"""What fused_attention must never use, though it lies inside a sequence: the
query rows that see no key (causal, more queries than keys) and the keys that
no query sees (below every row's window)."""
import pytest
import torch

import bloth_b200
from attention_reference import attention, check, sequences

pytestmark = pytest.mark.gpu

BF, FH, F32 = torch.bfloat16, torch.float16, torch.float32


def _run(dev, dtype, D, B, Sq, Sk, window=None, q_lens=None, k_lens=None, cu=None, cu_k=None,
         bad=float("nan"), backward=True):
    gen = torch.Generator(device=dev).manual_seed(Sq * 1000 + Sk)
    rand = lambda s, h: torch.randn(B, s, h, D, generator=gen, device=dev).to(dtype)  # noqa: E731
    q, do, k, v = rand(Sq, 4), rand(Sq, 4), rand(Sk, 2), rand(Sk, 2)
    seqs = sequences(B, Sq, Sk, q_lens, k_lens, cu, cu_k)
    want = attention(q, k, v, do, seqs, True, window)
    rows = 0
    for b, q0, nq, k0, nk in seqs:
        none = max(0, nq - nk)  # queries before the first key
        for x in (q, do):
            x[b, q0:q0 + none] = bad
        below = max(0, nk - nq - window + 1) if window else 0
        for x in (k, v):
            x[b, k0:k0 + below] = bad
        rows += none + below
    assert rows > 0
    t = lambda x: x and torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    call = lambda: bloth_b200.fused_attention(  # noqa: E731
        q, k, v, window=window, q_lens=t(q_lens), k_lens=t(k_lens), cu_seqlens=t(cu),
        cu_seqlens_k=t(cu_k))
    check(call(), want["o"], "o without gradients")
    if not backward:
        return
    for x in (q, k, v):
        x.requires_grad_(True)
    o = call()
    check(o.detach(), want["o"], "o")
    for n, x in zip(("dq", "dk", "dv"), torch.autograd.grad(o, (q, k, v), do)):
        check(x, want[n], n)
    assert bloth_b200.device_fault() == 0


TYPES = [(BF, 64), (BF, 128), (BF, 256), (FH, 64), (FH, 128), (F32, 64), (F32, 256)]


@pytest.mark.parametrize("dtype,D", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("Sq,Sk", [(300, 130), (300, 1), (257, 250), (100, 37)])
def test_queries_before_the_first_key(cuda, dtype, D, bad, Sq, Sk):
    _run(cuda, dtype, D, 2, Sq, Sk, bad=bad)


@pytest.mark.parametrize("dtype,D", TYPES)
def test_queries_before_the_first_key_of_some_sequences(cuda, dtype, D):
    _run(cuda, dtype, D, 4, 200, 200, q_lens=[200, 150, 70, 5], k_lens=[137, 200, 1, 0])
    _run(cuda, dtype, D, 1, 300, 300, cu=[0, 100, 170, 300], cu_k=[0, 33, 200, 300])


@pytest.mark.parametrize("dtype,D", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("Sq,Sk,window", [(150, 333, 50), (300, 700, 5), (129, 200, 70),
                                          (40, 500, 300)])
def test_keys_below_every_window(cuda, dtype, D, bad, Sq, Sk, window):
    _run(cuda, dtype, D, 2, Sq, Sk, window, bad=bad)


@pytest.mark.parametrize("dtype,D", TYPES)
@pytest.mark.parametrize("Sq,window", [(1, 7), (1, 300), (3, 100), (7, 1)])
def test_cached_keys_below_the_window_of_a_few_rows(cuda, dtype, D, Sq, window):
    _run(cuda, dtype, D, 3, Sq, 900, window, k_lens=[900, 333, 650], backward=Sq == 3)


@pytest.mark.parametrize("dtype,D", TYPES)
def test_keys_below_every_window_of_packed_sequences(cuda, dtype, D):
    _run(cuda, dtype, D, 1, 400, 900, 30, cu=[0, 10, 200, 400], cu_k=[0, 200, 600, 900])
