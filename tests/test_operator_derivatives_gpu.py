"""Derivatives that the attention and multi-axis rotary operators do not have
are refused, not dropped: second ones, and forward-mode ones."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

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


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_derivatives_are_refused(cuda, name, grad):
    x, f = _calls(cuda)[name]
    for i in range(len(x)):
        with fwad.dual_level(), torch.set_grad_enabled(grad):
            y = list(x)
            y[i] = fwad.make_dual(x[i], torch.ones_like(x[i]))
            with pytest.raises((RuntimeError, NotImplementedError)):
                f(*y)


def test_forward_mode_derivatives_by_frequency_are_refused(cuda):
    q = torch.randn(1, 6, 2, 64, device=cuda)
    pos, inv = torch.arange(6, device=cuda).expand(3, 1, 6), torch.ones(32, device=cuda)
    with fwad.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        bloth_b200.apply_mrope_qk(q, None, pos, fwad.make_dual(inv, inv.clone()),
                                  bloth_b200.mrope_axes((12, 10, 10)))


@pytest.mark.parametrize("name", NAMES)
def test_plain_tensors_inside_a_dual_level(cuda, name):
    x, f = _calls(cuda)[name]
    want = f(*x)
    with fwad.dual_level():
        assert torch.equal(f(*x), want)
