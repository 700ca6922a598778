"""Layouts and arguments of the attention and multi-axis rotary operators that
no address depends on, or that come in other types than each other."""
import pytest
import torch

import bloth_b200

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _odd(x):
    """x with an odd stride in each dimension of one element."""
    st = [7 if n == 1 and i < x.dim() - 1 else s for i, (n, s) in enumerate(zip(x.shape, x.stride()))]
    return x.as_strided(x.shape, st)


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("B,S,Hq,Hk", [(1, 40, 4, 2), (2, 1, 4, 1), (1, 1, 1, 1), (1, 300, 1, 1)])
def test_strides_of_single_elements(cuda, dtype, B, S, Hq, Hk):
    gen = torch.Generator(device=cuda).manual_seed(1)
    q, do = (torch.randn(B, S, Hq, 64, generator=gen, device=cuda).to(dtype) for _ in range(2))
    k, v = (torch.randn(B, S, Hk, 64, generator=gen, device=cuda).to(dtype) for _ in range(2))
    pos = torch.arange(S, device=cuda).expand(2, 1, S)
    w = torch.ones(64, device=cuda, dtype=dtype)
    inv, axes = torch.ones(32, device=cuda), bloth_b200.mrope_axes((16, 16))

    def run(q, k, v, do):
        q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
        o = bloth_b200.fused_attention(q, k, v)
        r = bloth_b200.apply_mrope_qk(q, k, pos, inv, axes)
        n = bloth_b200.fused_qk_norm_mrope(q, k, w, w, pos, inv, axes)
        m = bloth_b200.fused_qk_norm_rope(q, k, w, w, pos[0], inv)
        return (o, *torch.autograd.grad(o, (q, k, v), do), *r, *n, *m,
                *torch.autograd.grad(n[0], q, do))

    for a, b in zip(run(q, k, v, do), run(*(_odd(x) for x in (q, k, v, do)))):
        assert torch.equal(a, b)


def test_offsets_of_two_types(cuda):
    # 64-bit offsets beside 32-bit ones keep their value: past the keys' end here
    gen = torch.Generator(device=cuda).manual_seed(2)
    q, k, v = (torch.randn(100, h, 64, generator=gen, device=cuda).to(BF) for h in (2, 1, 1))
    t = lambda x, d: torch.tensor(x, device=cuda, dtype=d)  # noqa: E731
    far = [0, 30, 2 ** 32 + 60]
    want = bloth_b200.fused_attention(q, k, v, cu_seqlens=t([0, 50, 100], torch.int64),
                                      cu_seqlens_k=t([0, 30, 100], torch.int64))
    for d in (torch.int32, torch.int64):
        assert torch.equal(want, bloth_b200.fused_attention(
            q, k, v, cu_seqlens=t([0, 50, 100], d), cu_seqlens_k=t(far, torch.int64)))
    want = bloth_b200.fused_attention(q, k, v, cu_seqlens=t([0, 30, 100], torch.int64),
                                      cu_seqlens_k=t([0, 50, 100], torch.int64))
    assert torch.equal(want, bloth_b200.fused_attention(
        q, k, v, cu_seqlens=t(far, torch.int64), cu_seqlens_k=t([0, 50, 100], torch.int32)))
