"""Layouts of the attention and rotary operators that no address depends on."""
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
