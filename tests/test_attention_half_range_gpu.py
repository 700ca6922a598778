"""fp16 attention where probabilities leave fp16's normal range (from 2^-14) and
the results do not."""
import math

import pytest
import torch

import bloth_b200

pytestmark = pytest.mark.gpu

FH = torch.float16
U, T = 2.0 ** -11, 2.0 ** -25


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
