"""fp16 attention where probabilities and ds leave fp16's normal range
(2^-14 to 65504) and the results do not. The bounds are attention_reference.py's
with the unit roundoff of fp16 and no loss for small numbers: `inner` is fp16's
roundoff on fp32 copies of the inputs, plus the results' own rounding."""
import math

import pytest
import torch

import bloth_b200
from attention_reference import attention, check, sequences

pytestmark = pytest.mark.gpu

FH = torch.float16
U, T = 2.0 ** -11, 2.0 ** -25


def _run(dev, D, B, Sq, Sk, sizes, causal=True, few=False, rows=None, names=None, Hq=2, Hk=1,
         **kw):
    """sizes: of q, k, v, do; rows: factors of do's rows."""
    gen = torch.Generator(device=dev).manual_seed(D + Sq + Sk)
    rand = lambda s, h, a: (torch.randn(B, s, h, D, generator=gen, device=dev) * a)  # noqa: E731
    q, k, v, do = (rand(s, h, a) for s, h, a in zip((Sq, Sk, Sk, Sq), (Hq, Hk, Hk, Hq), sizes))
    if rows is not None:
        do *= rows.view(1, -1, 1, 1)
    q, k, v, do = (x.to(FH) for x in (q, k, v, do))
    assert all(torch.isfinite(x).all() for x in (q, k, v, do))
    cu = kw.get("cu")
    want = attention(q.float(), k.float(), v.float(), do.float(), sequences(B, Sq, Sk, cu_q=cu),
                     causal, inner=U ** 2 if few else U)
    q, k, v = (x.requires_grad_(True) for x in (q, k, v))
    o = bloth_b200.fused_attention(
        q, k, v, causal=causal,
        cu_seqlens=cu and torch.tensor(cu, dtype=torch.int32, device=dev))
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(o, (q, k, v), do)), o=o.detach())
    assert bloth_b200.device_fault() == 0
    for n in names or got:
        val, err = want[n]
        assert float(val.abs().max()) < 65504
        check(got[n], (val, err + U * val.abs() + T), n)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_probabilities_of_many_keys(cuda, D):
    # p = 1 / 138000 = 121.6 * 2^-24: rounded to fp16 as it is, off by 0.35%
    Sq, Sk = 130, 138000
    gen = torch.Generator(device=cuda).manual_seed(D)
    q, v = torch.zeros(1, Sq, 1, D, device=cuda), torch.ones(1, Sk, 1, D, device=cuda)
    k = torch.randn(1, Sk, 1, D, generator=gen, device=cuda)
    do = 50 + 100 * torch.rand(1, Sq, 1, D, generator=gen, device=cuda)
    q, k, v, do = (x.to(FH) for x in (q, k, v, do))
    v.requires_grad_(True)
    dv, = torch.autograd.grad(bloth_b200.fused_attention(q, k, v, causal=False), v, do)
    assert bloth_b200.device_fault() == 0
    want = (do.double().sum(1) / Sk).unsqueeze(1)
    # p's rounding and dv's, an fp32 sum of Sk / 64 blocks, one of Sq products,
    # the exponential's 64 roundings
    tol = (2 * U + (Sk // 64 + Sq + 66) * 2.0 ** -24) * want + T
    assert ((dv.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("Sq", [1, 8, 200])
def test_small_probabilities_beside_a_large_one(cuda, Sq):
    # key 0 has weight 1, each other 2^-20.47 = 11.6 * 2^-24: rounded to fp16 as
    # it is, off by 3.7%; v of key 0 is zero, so that the others are the result
    D, n = 64, 16384
    q, v = torch.zeros(1, Sq, 1, D, device=cuda), torch.ones(1, n, 1, D, device=cuda)
    k = torch.zeros(1, n, 1, D, device=cuda)
    q[..., 0], k[0, 0, 0, 0], v[0, 0] = 8.0, 20.47 * math.log(2.0), 0.0
    q, k, v = (x.to(FH) for x in (q, k, v))
    w = torch.exp(k.double()[0, :, 0, 0])  # scale is 1/8
    want = float(w[1:].sum() / w.sum())
    got = bloth_b200.fused_attention(q, k, v, causal=False).double()
    # p's rounding and the result's, an fp32 sum of n terms, the exponential
    assert float((got - want).abs().max()) <= (2 * U + (n + 66) * 2.0 ** -24) * want


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Sk,few", [(5, True), (300, False)])
@pytest.mark.parametrize("causal", [True, False])
def test_large_ds(cuda, D, Sk, few, causal):
    # dp around 2^23, p around 1/300: ds above 65504
    _run(cuda, D, 2, Sk, Sk, (0.004, 0.004, 200.0, 4000.0), causal, few)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Sk,few", [(100, True), (700, False)])
@pytest.mark.parametrize("causal", [True, False])
def test_small_ds(cuda, D, Sk, few, causal):
    # dp around 2^-17, p around 1/700: ds below 2^-25; dq a thousand times larger
    _run(cuda, D, 1, Sk, Sk, (1e-4, 8000.0, 0.01, 1e-4), causal, few, names=("dq",))
    # and dk
    _run(cuda, D, 1, Sk, Sk, (8000.0, 1e-4, 0.01, 1e-4), causal, few, names=("dk",))


@pytest.mark.parametrize("D", [64, 128, 256])
def test_ds_of_documents_of_different_sizes(cuda, D):
    cu = [0, 300, 700, 1000]
    rows = torch.ones(1000, device=cuda)
    rows[300:700], rows[700:] = 2.0 ** 20, 2.0 ** 10
    _run(cuda, D, 1, 1000, 1000, (1e-4, 300.0, 0.01, 1e-3), rows=rows, cu=cu, names=("dq",))
    _run(cuda, D, 1, 1000, 1000, (300.0, 1e-4, 0.01, 1e-3), rows=rows, cu=cu, names=("dk",))


@pytest.mark.parametrize("D", [64, 128])
def test_dq_of_rows_of_different_sizes(cuda, D):
    # a row's ds have a range of their own in dq
    rows = 2.0 ** torch.randint(-10, 20, (400,), device=cuda).float()
    _run(cuda, D, 1, 400, 400, (1e-4, 300.0, 0.01, 1e-3), rows=rows, names=("dq",))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Sq,Sk,few", [(5, 5, True), (300, 300, False), (4, 700, False)])
def test_delta_of_small_outputs(cuda, D, Sq, Sk, few):
    # o below fp16's normal range: what its rounding takes off is at most 2^-25
    _run(cuda, D, 1, Sq, Sk, (1.0, 1.0, 2e-6, 3000.0), few=few, names=("dq", "dk"))
