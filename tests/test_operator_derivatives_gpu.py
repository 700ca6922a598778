"""Derivatives that the attention and multi-axis rotary operators do not have
are refused, not dropped."""
import pytest
import torch

import bloth_b200

pytestmark = pytest.mark.gpu


def _calls(dev):
    q, k, v = (torch.randn(1, 6, h, 64, device=dev) for h in (2, 1, 1))
    pos = torch.arange(6, device=dev).expand(3, 1, 6)
    inv = torch.ones(32, device=dev)
    axes = bloth_b200.mrope_axes((12, 10, 10))
    w = torch.ones(64, device=dev)
    return {
        "attention": ((q, k, v), lambda q, k, v: bloth_b200.fused_attention(q, k, v)),
        "lse": ((q, k, v), lambda q, k, v: bloth_b200.fused_attention(q, k, v, return_lse=True)[0]),
        "mrope": ((q, k), lambda q, k: bloth_b200.apply_mrope_qk(q, k, pos, inv, axes)[0]),
        "norm": ((q, k, w, w.clone()), lambda q, k, a, b: bloth_b200.fused_qk_norm_mrope(
            q, k, a, b, pos, inv, axes)[0]),
    }


NAMES = ["attention", "lse", "mrope", "norm"]


@pytest.mark.parametrize("name", NAMES)
def test_second_derivatives_are_refused(cuda, name):
    x, f = _calls(cuda)[name]
    x = [t.requires_grad_(True) for t in x]
    g, = torch.autograd.grad(f(*x).square().sum(), x[0], create_graph=True)
    # another path keeps the penalty differentiable
    with pytest.raises(RuntimeError, match="once_differentiable"):
        (g.square().sum() + x[0].sum()).backward()
