"""Rotary positions with several axes against a plain 64-bit implementation.

Tolerances, element for element, with u the unit roundoff of the tensors' type
and w = 2^-24: an output is a sum of two products of a normalised value (at
most a few w relative: squares, mean, rsqrt and weight), with cos and sin good
to 2 ulp, so |err| <= u |y| + 32 w (|n1| + |n2|); gradients alike, with sums
over a row (D terms) for dx and over all rows for the weights.
"""
import pytest
import torch

import bloth_b200

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
W = 2.0 ** -24
BF, FH, F32 = torch.bfloat16, torch.float16, torch.float32


def _turn(x, cos, sin, back=False):
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    if back:
        sin = -sin
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _size(x):
    """|x1| + |x2| of each pair, at both of its places."""
    h = x.shape[-1] // 2
    s = x[..., :h].abs() + x[..., h:].abs()
    return torch.cat([s, s], -1)


def _reference(x, g, w, pos, inv_freq, axes, eps, offset, scale):
    """(y, dx, dw) and their bounds for one [B, S, H, D] tensor."""
    D = x.shape[-1]
    p = pos if pos.dim() == 3 else pos.unsqueeze(1)
    p = p.expand(p.shape[0], x.shape[0], x.shape[1])
    ang = (p[list(axes)].permute(1, 2, 0).float() * inv_freq).double()
    cos, sin = (scale * f(ang).unsqueeze(2) for f in (torch.cos, torch.sin))
    u, xd, gd = U[x.dtype], x.double(), g.double()
    if w is None:
        y, dx = _turn(xd, cos, sin), _turn(gd, cos, sin, True)
        return ((y, u * y.abs() + 32 * W * scale * _size(xd)),
                (dx, u * dx.abs() + 32 * W * scale * _size(gd)), None)
    wd = w.double() + offset
    rstd = (xd.square().mean(-1, keepdim=True) + eps).rsqrt()
    xh = xd * rstd
    r = (D + 16) * W  # relative error of rstd and of row sums
    y = _turn(xh * wd, cos, sin)
    dn = _turn(gd, cos, sin, True)
    dne = 32 * W * scale * _size(gd)
    t = dn * wd
    te = dne * wd.abs() + 4 * W * t.abs()
    mean = (t * xh).mean(-1, keepdim=True)
    me = (te * xh.abs() + 2 * r * (t * xh).abs()).mean(-1, keepdim=True)
    dx = rstd * (t - xh * mean)
    dxe = rstd * (te + xh.abs() * (me + r * mean.abs()) + r * (t.abs() + (xh * mean).abs()))
    dw = (dn * xh).sum((0, 1, 2))
    rows = x.shape[0] * x.shape[1] * x.shape[2]
    # per-thread sums, folded: at most `rows` additions (fp64 for fp32 tensors)
    acc = W * (rows if x.dtype != F32 else 4)
    dwe = (dne * xh.abs() + (r + acc) * (dn * xh).abs()).sum((0, 1, 2)) + U[w.dtype] * dw.abs()
    return ((y, u * y.abs() + (32 * W + r) * scale * _size(xh * wd)),
            (dx, u * dx.abs() + dxe), (dw, dwe))


def _check(got, want, name):
    val, err = want
    tiny = 2.0 ** -24 if got.dtype == FH else 1e-38
    off = (got.double() - val).abs() - err
    assert float(off.max()) <= tiny, f"{name}: off by {float(off.max()):.3e} beyond the bound"


def _positions(A, B, S, gen, dev, dtype=torch.int64, top=4000):
    return torch.randint(0, top, (A, B, S), generator=gen, device=dev).to(dtype)


def _run(dev, dtype, D, B, S, Hq, Hk, sections, interleaved=False, norm=True, heads_first=False,
         pos_dtype=torch.int64, offset=0.0, scale=1.0, w_dtype=None, seed=0):
    gen = torch.Generator(device=dev).manual_seed(seed)

    def mk(h):
        if heads_first:
            return torch.randn(B, h, S, D, generator=gen, device=dev).to(dtype).transpose(1, 2)
        return torch.randn(B, S, h, D, generator=gen, device=dev).to(dtype)

    q, k, gq, gk = mk(Hq), mk(Hk), mk(Hq), mk(Hk)
    wq, wk = ((1 + 0.2 * torch.randn(D, generator=gen, device=dev)).to(w_dtype or dtype)
              for _ in range(2))
    pos = _positions(len(sections), B, S, gen, dev, pos_dtype)
    inv = 1.0 / (1e4 ** (torch.arange(D // 2, device=dev, dtype=F32) / (D // 2)))
    axes = bloth_b200.mrope_axes(sections, interleaved)
    ins = [t.requires_grad_(True) for t in ((q, k, wq, wk) if norm else (q, k))]
    if norm:
        out = bloth_b200.fused_qk_norm_mrope(q, k, wq, wk, pos, inv, axes, eps=1e-6,
                                             weight_offset=offset, rope_scale=scale)
    else:
        out = bloth_b200.apply_mrope_qk(q, k, pos, inv, axes, rope_scale=scale)
    grads = torch.autograd.grad(out, ins, [gq, gk])
    assert bloth_b200.device_fault() == 0
    for i, (x, g, w) in enumerate(((q, gq, wq), (k, gk, wk))):
        y, dx, dw = _reference(x.detach(), g, w.detach() if norm else None, pos, inv, axes, 1e-6,
                               offset, scale)
        n = "qk"[i]
        _check(out[i].detach(), y, n)
        _check(grads[i], dx, "d" + n)
        if norm:
            _check(grads[2 + i], dw, "dw" + n)
    return out, grads


SECTIONS = {64: ([8, 12, 12], [12, 10, 10]), 128: ([16, 24, 24], [24, 20, 20]),
            256: ([32, 48, 48], [48, 40, 40])}


@pytest.mark.parametrize("dtype", [BF, FH, F32])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("interleaved", [False, True])
def test_types_and_head_dims(cuda, dtype, D, norm, interleaved):
    _run(cuda, dtype, D, 2, 77, 8, 4, SECTIONS[D][interleaved], interleaved, norm)


@pytest.mark.parametrize("S", [1, 2, 31, 300])
@pytest.mark.parametrize("Hq,Hk", [(4, 4), (5, 1), (32, 8), (1, 3)])
def test_lengths_and_heads(cuda, S, Hq, Hk):
    _run(cuda, BF, 128, 1, S, Hq, Hk, [16, 24, 24], seed=S)
    _run(cuda, BF, 64, 3, S, Hq, Hk, [12, 10, 10], True, norm=False, seed=S)


@pytest.mark.parametrize("sections", [[64], [40, 24], [16, 24, 24], [10, 18, 18, 18], [0, 32, 32]])
def test_one_to_four_axes(cuda, sections):
    _run(cuda, BF, 128, 2, 50, 4, 4, sections)
    _run(cuda, F32, 128, 2, 50, 4, 2, sections, norm=False)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_layouts_positions_and_scales(cuda, dtype):
    _run(cuda, dtype, 128, 2, 90, 6, 2, [16, 24, 24], heads_first=True)
    _run(cuda, dtype, 64, 2, 90, 6, 2, [8, 12, 12], norm=False, heads_first=True)
    _run(cuda, dtype, 64, 2, 90, 4, 4, [8, 12, 12], pos_dtype=torch.int32)
    _run(cuda, dtype, 128, 2, 90, 4, 4, [16, 24, 24], offset=1.0, scale=1.25, w_dtype=F32)


def test_many_tokens(cuda):
    # beyond one wave of CTAs, and beyond the forward's token-block kernel
    _run(cuda, BF, 64, 3, 3001, 8, 4, [12, 10, 10], True)


def test_shapes_of_positions(cuda):
    gen = torch.Generator(device=cuda).manual_seed(1)
    q, k = (torch.randn(2, 40, h, 64, generator=gen, device=cuda).to(BF) for h in (4, 2))
    inv = 1.0 / (1e4 ** (torch.arange(32, device=cuda, dtype=F32) / 32))
    axes = bloth_b200.mrope_axes([8, 12, 12])
    one = _positions(3, 1, 40, gen, cuda)
    want = bloth_b200.apply_mrope_qk(q, k, one.expand(3, 2, 40).contiguous(), inv, axes)
    wide = torch.full((3, 2, 80), 7, device=cuda)
    wide[:, :, ::2] = one
    for pos in (one, one[:, 0], one.expand(3, 2, 40), wide[:, :, ::2]):
        got = bloth_b200.apply_mrope_qk(q, k, pos, inv, axes)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # three-dimensional tensors, and q alone
    got = bloth_b200.apply_mrope_qk(q[0], None, one, inv, axes)
    assert torch.equal(got, want[0][0])
    w = torch.ones(64, device=cuda, dtype=BF)
    alone = bloth_b200.fused_qk_norm_mrope(q, None, w, None, one, inv, axes)
    both = bloth_b200.fused_qk_norm_mrope(q, k, w, w, one, inv, axes)
    assert torch.equal(alone, both[0])


@pytest.mark.parametrize("norm", [True, False])
def test_equal_axes_are_one_position(cuda, norm):
    gen = torch.Generator(device=cuda).manual_seed(2)
    q, k = (torch.randn(2, 100, h, 128, generator=gen, device=cuda).to(BF) for h in (8, 4))
    w = torch.ones(128, device=cuda, dtype=BF)
    inv = 1.0 / (1e4 ** (torch.arange(64, device=cuda, dtype=F32) / 64))
    pos = torch.randint(0, 9999, (2, 100), generator=gen, device=cuda)
    axes = bloth_b200.mrope_axes([16, 24, 24])
    if norm:
        a = bloth_b200.fused_qk_norm_rope(q, k, w, w, pos, inv)
        b = bloth_b200.fused_qk_norm_mrope(q, k, w, w, pos.expand(3, 2, 100), inv, axes)
    else:
        a = bloth_b200.apply_rope_qk(q, k, pos, inv)
        b = bloth_b200.apply_mrope_qk(q, k, pos.expand(3, 2, 100), inv, axes)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_gradients_against_differences(cuda):
    gen = torch.Generator(device=cuda).manual_seed(3)
    q, k = (torch.randn(1, 20, h, 64, generator=gen, device=cuda) for h in (4, 2))
    w = [1 + 0.2 * torch.randn(64, generator=gen, device=cuda) for _ in range(2)]
    pos = _positions(3, 1, 20, gen, cuda)
    inv = 1.0 / (1e4 ** (torch.arange(32, device=cuda, dtype=F32) / 32))
    axes = bloth_b200.mrope_axes([12, 10, 10], True)
    x = [q, k, *w]
    way = [torch.randn(t.shape, generator=gen, device=cuda) for t in x]
    g = [torch.randn(t.shape, generator=gen, device=cuda) for t in (q, k)]

    def at(h):
        y = bloth_b200.fused_qk_norm_mrope(*(a + h * b for a, b in zip(x, way)), pos, inv, axes)
        return float(sum((a.double() * b.double()).sum() for a, b in zip(y, g)))

    h = 2.0 ** -7  # fourth order: truncation O(h^4), roundoff sqrt(n) 2^-23 / h
    slope = (8 * (at(h) - at(-h)) - (at(2 * h) - at(-2 * h))) / (12 * h)
    leaves = [t.clone().requires_grad_(True) for t in x]
    grads = torch.autograd.grad(
        bloth_b200.fused_qk_norm_mrope(*leaves, pos, inv, axes), leaves, g)
    got = float(sum((a.double() * b.double()).sum() for a, b in zip(grads, way)))
    size = float(sum((a.double() * b.double()).square().sum() for a, b in zip(grads, way))) ** 0.5
    assert abs(got - slope) < 5e-3 * size, (got, slope, size)


def test_as_the_vision_language_models_do(cuda):
    """Against transformers' rotation with cos and sin laid out by section."""
    m2 = pytest.importorskip("transformers.models.qwen2_vl.modeling_qwen2_vl")
    gen = torch.Generator(device=cuda).manual_seed(4)
    q, k = (torch.randn(2, 33, h, 128, generator=gen, device=cuda) for h in (4, 2))
    pos = _positions(3, 2, 33, gen, cuda)
    inv = 1.0 / (1e6 ** (torch.arange(64, device=cuda, dtype=F32) / 64))
    ang = pos.float().unsqueeze(-1) * inv  # [3, B, S, 64]
    sec = [16, 24, 24]
    if not hasattr(m2, "apply_multimodal_rotary_pos_emb"):
        pytest.skip("this transformers version has no apply_multimodal_rotary_pos_emb")
    emb = torch.cat([ang, ang], -1)
    want = m2.apply_multimodal_rotary_pos_emb(q.transpose(1, 2), k.transpose(1, 2), emb.cos(),
                                              emb.sin(), sec)
    got = bloth_b200.apply_mrope_qk(q, k, pos, inv, bloth_b200.mrope_axes(sec))
    for a, b in zip(got, want):
        assert (a - b.transpose(1, 2)).abs().max() < 1e-5


def test_refusals(cuda):
    q = torch.randn(2, 8, 4, 64, device=cuda, dtype=BF)
    k = torch.randn(2, 8, 2, 64, device=cuda, dtype=BF)
    w = torch.ones(64, device=cuda, dtype=BF)
    pos = torch.zeros(3, 2, 8, device=cuda, dtype=torch.int64)
    inv = torch.ones(32, device=cuda)
    axes = bloth_b200.mrope_axes([8, 12, 12])
    f = bloth_b200.apply_mrope_qk
    for bad in ((q, k, pos[:, :, :7], inv, axes), (q, k, pos[:, :1].expand(3, 3, 8), inv, axes),
                (q, k, pos[0, 0], inv, axes), (q, k, pos.expand(3, 2, 8)[:0], inv, axes),
                (q, k, torch.zeros(5, 2, 8, device=cuda).long(), inv, axes),
                (q, k, pos, inv[:31], axes), (q, k, pos, inv, axes[:31]),
                (q, k, pos[:2], inv, axes), (q, k, pos, inv, (3,) * 32),
                (q, k, pos, inv, (-1,) * 32), (q, k[:, :7], pos, inv, axes)):
        with pytest.raises(ValueError):
            f(*bad)
    with pytest.raises(TypeError):
        f(q, k.float(), pos, inv, axes)
    with pytest.raises(ValueError):
        bloth_b200.fused_qk_norm_mrope(q, k, w, None, pos, inv, axes)
    with pytest.raises(ValueError):
        bloth_b200.fused_qk_norm_mrope(q, k, w, w[:32], pos, inv, axes)
    with pytest.raises(RuntimeError):
        f(q[..., :32].contiguous(), k[..., :32].contiguous(), pos, inv[:16], axes[:16])
    with pytest.raises(AssertionError, match="CUDA GPU required"):
        f(q.cpu(), k.cpu(), pos.cpu(), inv.cpu(), axes)
