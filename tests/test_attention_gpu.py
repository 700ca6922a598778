"""fused_attention and its backward against a plain 64-bit implementation
(attention_reference.py, which also derives the tolerances), at the sizes and
masks where tiles end, start empty or see nothing."""
import pytest
import torch

import bloth_b200
from attention_reference import attention, check, sequences

pytestmark = pytest.mark.gpu

BF, FH, F32 = torch.bfloat16, torch.float16, torch.float32


def _rand(shape, dtype, gen, dev, heads_first=False):
    if heads_first:
        b, s, h, d = shape
        return torch.randn(b, h, s, d, generator=gen, device=dev).to(dtype).transpose(1, 2)
    return torch.randn(*shape, generator=gen, device=dev).to(dtype)


def _run(dev, dtype, D, B, Sq, Sk, Hq, Hk, causal=True, window=None, scale=None, q_lens=None,
         k_lens=None, cu=None, cu_k=None, heads_first=False, seed=0, index=torch.int32,
         poison=False):
    gen = torch.Generator(device=dev).manual_seed(seed)
    q, do = (_rand((B, Sq, Hq, D), dtype, gen, dev, heads_first) for _ in range(2))
    k, v = (_rand((B, Sk, Hk, D), dtype, gen, dev, heads_first) for _ in range(2))
    seqs = sequences(B, Sq, Sk, q_lens, k_lens, cu, cu_k)
    want = attention(q, k, v, do, seqs, causal, window, scale)
    if poison:  # whatever lies outside of the sequences is never used
        for x, at, n in ((q, 1, 2), (do, 1, 2), (k, 3, 4), (v, 3, 4)):
            inside = torch.zeros(x.shape[:2], dtype=torch.bool, device=dev)
            for s in seqs:
                inside[s[0], s[at]:s[at] + s[n]] = True
            x[~inside] = float("nan")
    t = lambda x: None if x is None else torch.tensor(x, dtype=index, device=dev)  # noqa: E731
    q, k, v = (x.requires_grad_(True) for x in (q, k, v))
    o, lse = bloth_b200.fused_attention(q, k, v, causal=causal, window=window, scale=scale,
                                        q_lens=t(q_lens), k_lens=t(k_lens), cu_seqlens=t(cu),
                                        cu_seqlens_k=t(cu_k), return_lse=True)
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), do)
    torch.cuda.synchronize()
    assert bloth_b200.device_fault() == 0
    got = {"o": o, "lse": lse, "dq": dq, "dk": dk, "dv": dv}
    for n, x in got.items():
        assert x.dtype == (F32 if n == "lse" else dtype)
        check(x.detach(), want[n], n)
    # the form without gradients gives the same rows
    with torch.no_grad():
        again = bloth_b200.fused_attention(q, k, v, causal=causal, window=window, scale=scale,
                                           q_lens=t(q_lens), k_lens=t(k_lens), cu_seqlens=t(cu),
                                           cu_seqlens_k=t(cu_k))
    check(again, want["o"], "o without gradients")
    return got


@pytest.mark.parametrize("dtype", [BF, FH, F32])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_types_and_head_dims(cuda, dtype, D, causal):
    _run(cuda, dtype, D, 2, 200, 200, 4, 2, causal)


@pytest.mark.parametrize("dtype,D", [(BF, 128), (FH, 64), (F32, 64), (BF, 256)])
@pytest.mark.parametrize("S", [1, 2, 63, 64, 65, 127, 128, 129, 255, 256, 257, 513])
def test_lengths(cuda, dtype, D, S):
    _run(cuda, dtype, D, 1, S, S, 3, 1, seed=S)


@pytest.mark.parametrize("dtype,D", [(BF, 128), (FH, 64), (F32, 128)])
@pytest.mark.parametrize("Sq,Sk", [(1, 1000), (3, 129), (17, 640), (128, 700), (300, 1100)])
def test_chunk_after_a_cache(cuda, dtype, D, Sq, Sk):
    _run(cuda, dtype, D, 2, Sq, Sk, 8, 2, seed=Sq)


@pytest.mark.parametrize("dtype,D", [(BF, 128), (FH, 64), (F32, 64)])
@pytest.mark.parametrize("Sq,Sk", [(300, 1), (300, 130), (257, 256), (1000, 3)])
def test_more_queries_than_keys(cuda, dtype, D, Sq, Sk):
    # causal: the first Sq - Sk rows see nothing
    got = _run(cuda, dtype, D, 2, Sq, Sk, 4, 2, seed=Sk)
    assert (got["o"][:, :Sq - Sk] == 0).all() and (got["dq"][:, :Sq - Sk] == 0).all()
    _run(cuda, dtype, D, 1, Sq, Sk, 4, 2, causal=False, seed=Sk)


@pytest.mark.parametrize("dtype,D", [(BF, 128), (FH, 64), (F32, 64), (BF, 64)])
@pytest.mark.parametrize("window", [1, 5, 64, 100, 128, 300, 10 ** 12])
def test_window(cuda, dtype, D, window):
    _run(cuda, dtype, D, 1, 400, 400, 2, 1, window=window)
    _run(cuda, dtype, D, 1, 150, 333, 2, 1, window=window)


@pytest.mark.parametrize("Hq,Hk", [(1, 1), (5, 5), (7, 1), (12, 4), (32, 8)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_head_groups(cuda, dtype, Hq, Hk):
    _run(cuda, dtype, 64, 2, 140, 140, Hq, Hk, seed=Hq)


@pytest.mark.parametrize("dtype,D", [(BF, 128), (FH, 64), (F32, 64), (BF, 256)])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_padded_batch(cuda, dtype, D, index):
    lens = [0, 1, 77, 128, 200, 300]
    _run(cuda, dtype, D, 6, 300, 300, 4, 2, q_lens=lens, k_lens=lens, index=index, poison=True)
    _run(cuda, dtype, D, 6, 300, 300, 4, 2, causal=False, q_lens=lens, k_lens=lens, index=index,
         poison=True)


@pytest.mark.parametrize("dtype,D", [(BF, 128), (FH, 64), (F32, 64)])
def test_caches_in_use_up_to_a_length(cuda, dtype, D):
    for Sq in (1, 5, 40):
        _run(cuda, dtype, D, 5, Sq, 700, 8, 2, k_lens=[700, 40, 129, 300, 0], poison=True)


@pytest.mark.parametrize("dtype,D", [(BF, 128), (FH, 64), (F32, 64), (BF, 256), (BF, 64)])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_documents(cuda, dtype, D, causal):
    cu = [0, 0, 1, 130, 130, 258, 600, 601, 640]
    _run(cuda, dtype, D, 1, 640, 640, 4, 2, causal, cu=cu)
    # offsets that leave rows out at both ends: zeros there, and nothing read
    _run(cuda, dtype, D, 1, 640, 640, 4, 2, causal, cu=[3, 100, 333, 500], poison=True)


def test_many_packed_documents(cuda):
    cu = [0]
    for i in range(150):
        cu.append(cu[-1] + i % 7)
    _run(cuda, BF, 64, 1, cu[-1], cu[-1], 2, 1, cu=cu)


@pytest.mark.parametrize("dtype,D", [(BF, 128), (F32, 64)])
def test_packed_documents_with_their_own_keys(cuda, dtype, D):
    _run(cuda, dtype, D, 1, 400, 900, 4, 1, cu=[0, 10, 10, 300, 400], cu_k=[0, 200, 300, 301, 900],
         index=torch.int64)
    _run(cuda, dtype, D, 1, 400, 900, 4, 1, window=50, cu=[0, 10, 10, 300, 400],
         cu_k=[0, 200, 300, 301, 900])


@pytest.mark.parametrize("dtype", [BF, FH, F32])
def test_large_scores(cuda, dtype):
    # scores of +-100 and more: one key takes each row, running maxima move late
    _run(cuda, dtype, 64, 1, 300, 300, 2, 2, scale=4.0)
    _run(cuda, dtype, 128, 1, 300, 300, 2, 2, causal=False, scale=1e-3)


@pytest.mark.parametrize("dtype,D", [(BF, 128), (FH, 64), (F32, 256)])
def test_layouts(cuda, dtype, D):
    _run(cuda, dtype, D, 2, 150, 150, 4, 2, heads_first=True)
    # slices of one packed projection, and a gradient that repeats a row
    gen = torch.Generator(device=cuda).manual_seed(5)
    qkv = torch.randn(2, 150, 8, D, generator=gen, device=cuda).to(dtype)
    q, k, v = (x.detach().requires_grad_(True) for x in (qkv[:, :, :4], qkv[:, :, 4:6],
                                                         qkv[:, :, 6:]))
    do = torch.randn(1, 1, 1, D, generator=gen, device=cuda).to(dtype).expand(2, 150, 4, D)
    want = attention(q.detach(), k.detach(), v.detach(), do, sequences(2, 150, 150))
    o = bloth_b200.fused_attention(q, k, v)
    for n, x in zip(("o", "dq", "dk", "dv"), (o.detach(), *torch.autograd.grad(o, (q, k, v), do))):
        check(x, want[n], n)


def test_broadcast_keys_and_unaligned_rows(cuda):
    gen = torch.Generator(device=cuda).manual_seed(6)
    q = torch.randn(2, 70, 4, 64, generator=gen, device=cuda).to(BF).requires_grad_(True)
    one = torch.randn(1, 70, 1, 64, generator=gen, device=cuda).to(BF).requires_grad_(True)
    odd = torch.randn(2, 70, 4, 65, generator=gen, device=cuda).to(BF)[..., 1:]  # rows of 130 bytes
    do = torch.randn(2, 70, 4, 64, generator=gen, device=cuda).to(BF)
    k = one.expand(2, 70, 4, 64)
    o = bloth_b200.fused_attention(q, k, odd)
    dq, dk = torch.autograd.grad(o, (q, one), do)
    want = attention(q.detach(), k.detach(), odd, do, sequences(2, 70, 70))
    check(o.detach(), want["o"], "o")
    check(dq, want["dq"], "dq")
    val, err = want["dk"]
    # the eight copies' gradients, each rounded, are summed by autograd in bf16
    val, err = val.sum((0, 2)), err.sum((0, 2)) + 8 * 2.0 ** -8 * val.abs().sum((0, 2))
    check(dk[0, :, 0], (val, err), "dk")


def test_three_dimensional_tensors(cuda):
    gen = torch.Generator(device=cuda).manual_seed(7)
    q, k, v = (torch.randn(90, h, 64, generator=gen, device=cuda).to(BF).requires_grad_(True)
               for h in (4, 2, 2))
    o, lse = bloth_b200.fused_attention(q, k, v, return_lse=True)
    assert o.shape == q.shape and lse.shape == (4, 90) and not lse.requires_grad
    do = torch.randn(90, 4, 64, generator=gen, device=cuda).to(BF)
    want = attention(*(x.detach().unsqueeze(0) for x in (q, k, v)), do.unsqueeze(0),
                     sequences(1, 90, 90))
    check(o.detach().unsqueeze(0), want["o"], "o")
    for n, x in zip(("dq", "dk", "dv"), torch.autograd.grad(o, (q, k, v), do)):
        check(x.unsqueeze(0), want[n], n)


def test_gradients_of_some_inputs(cuda):
    gen = torch.Generator(device=cuda).manual_seed(8)
    mk = lambda h: torch.randn(1, 130, h, 64, generator=gen, device=cuda).to(BF)  # noqa: E731
    q, k, v, do = mk(4), mk(2), mk(2), mk(4)
    want = attention(q, k, v, do, sequences(1, 130, 130))
    for on in (("dq",), ("dk",), ("dv",), ("dq", "dv")):
        ins = {"dq": q.clone(), "dk": k.clone(), "dv": v.clone()}
        for n in on:
            ins[n].requires_grad_(True)
        o = bloth_b200.fused_attention(*ins.values())
        for n, x in zip(on, torch.autograd.grad(o, [ins[n] for n in on], do)):
            check(x, want[n], n)


def test_nothing_to_do(cuda):
    for B, Sq, Sk in ((0, 4, 4), (2, 0, 5), (2, 5, 0), (1, 0, 0)):
        q = torch.randn(B, Sq, 4, 64, device=cuda).to(BF).requires_grad_(True)
        k, v = (torch.randn(B, Sk, 2, 64, device=cuda).to(BF).requires_grad_(True)
                for _ in range(2))
        o, lse = bloth_b200.fused_attention(q, k, v, return_lse=True)
        assert (o == 0).all() and (lse == -float("inf")).all()
        for x, y in zip((q, k, v), torch.autograd.grad(o, (q, k, v), torch.ones_like(o))):
            assert y.shape == x.shape and (y == 0).all()


def test_offsets_out_of_the_tensors_are_clamped(cuda):
    gen = torch.Generator(device=cuda).manual_seed(9)
    q, k, v = (torch.randn(100, h, 64, generator=gen, device=cuda).to(BF) for h in (2, 1, 1))
    cu = torch.tensor([-5, 40, 20, 10 ** 6], device=cuda, dtype=torch.int32)
    want = torch.tensor([0, 40, 40, 100], device=cuda, dtype=torch.int32)
    assert torch.equal(bloth_b200.fused_attention(q, k, v, cu_seqlens=cu),
                       bloth_b200.fused_attention(q, k, v, cu_seqlens=want))
    x = q.unsqueeze(0), k.unsqueeze(0), v.unsqueeze(0)
    far = torch.tensor([10 ** 6], device=cuda)
    assert torch.equal(bloth_b200.fused_attention(*x, q_lens=far, k_lens=far),
                       bloth_b200.fused_attention(*x))


@pytest.mark.parametrize("dtype,D", [(BF, 128), (FH, 64), (F32, 64)])
def test_the_same_call_gives_the_same_bits(cuda, dtype, D):
    a = _run(cuda, dtype, D, 2, 500, 500, 8, 2)
    b = _run(cuda, dtype, D, 2, 500, 500, 8, 2)
    for n in a:
        assert torch.equal(a[n], b[n]), n


def test_another_stream(cuda):
    gen = torch.Generator(device=cuda).manual_seed(11)
    q, k, v, do = (torch.randn(1, 1000, h, 128, generator=gen, device=cuda).to(BF)
                   for h in (8, 2, 2, 8))
    q, k, v = (x.requires_grad_(True) for x in (q, k, v))
    o = bloth_b200.fused_attention(q, k, v)
    want = (o, *torch.autograd.grad(o, (q, k, v), do))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = bloth_b200.fused_attention(q, k, v)
        got = (o, *torch.autograd.grad(o, (q, k, v), do))
    side.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_in_a_graph(cuda):
    gen = torch.Generator(device=cuda).manual_seed(12)
    q, k, v, do = (torch.randn(1, 300, h, 64, generator=gen, device=cuda).to(BF)
                   for h in (8, 2, 2, 8))
    q, k, v = (x.requires_grad_(True) for x in (q, k, v))

    def step():
        o = bloth_b200.fused_attention(q, k, v)
        return (o, *torch.autograd.grad(o, (q, k, v), do))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [x.detach().clone() for x in step()]
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for x in got:
        x.detach().fill_(7)
    g.replay()
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("D", [64, 128])
def test_gradients_against_differences(cuda, D):
    # the directional derivative of sum(o * do) from fp32 outputs at +-h
    gen = torch.Generator(device=cuda).manual_seed(13)
    x = [torch.randn(1, 60, h, D, generator=gen, device=cuda) for h in (4, 2, 2)]
    way = [torch.randn(t.shape, generator=gen, device=cuda) for t in x]
    do = torch.randn(1, 60, 4, D, generator=gen, device=cuda)
    h = 2.0 ** -7

    def at(step):
        o = bloth_b200.fused_attention(*(a + step * b for a, b in zip(x, way)))
        return float((o.double() * do.double()).sum())

    # fourth-order central difference: truncation O(h^4), roundoff about
    # sqrt(n) * 2^-22 / h in units of the outputs
    slope = (8 * (at(h) - at(-h)) - (at(2 * h) - at(-2 * h))) / (12 * h)
    leaves = [t.clone().requires_grad_(True) for t in x]
    grads = torch.autograd.grad(bloth_b200.fused_attention(*leaves), leaves, do)
    got = float(sum((g.double() * w.double()).sum() for g, w in zip(grads, way)))
    size = float(sum((g.double().square() * w.double().square()).sum()
                     for g, w in zip(grads, way))) ** 0.5
    assert abs(got - slope) < 5e-3 * size, (got, slope, size)


def test_refusals(cuda):
    q = torch.randn(2, 8, 4, 64, device=cuda, dtype=BF)
    k = torch.randn(2, 8, 2, 64, device=cuda, dtype=BF)
    f = bloth_b200.fused_attention
    cu = torch.tensor([0, 8], device=cuda, dtype=torch.int32)
    for bad in (dict(window=0), dict(window=4, causal=False), dict(scale=0.0), dict(scale=-1.0),
                dict(scale=float("inf")), dict(scale=float("nan")), dict(cu_seqlens=cu),
                dict(k_lens=cu[:1]), dict(q_lens=cu.view(1, 2)), dict(cu_seqlens_k=cu),
                dict(k_lens=cu, cu_seqlens=cu)):
        with pytest.raises(ValueError):
            f(q, k, k, **bad)
    with pytest.raises(ValueError):
        f(q[0], k[0], k[0], cu_seqlens=cu[:1])
    with pytest.raises(ValueError):
        f(q[0], k[0, :4], k[0, :4], cu_seqlens=cu)
    with pytest.raises(ValueError):
        f(q, k, k[:, :4])
    with pytest.raises(ValueError):
        f(q, k[:1], k[:1])
    with pytest.raises(ValueError):
        f(q[:, :, :3], k, k)
    with pytest.raises(ValueError):
        f(q[..., :32], k[..., :32], k[..., :32])
    with pytest.raises(ValueError):
        f(q, k[0], k[0])
    with pytest.raises(TypeError):
        f(q, k.float(), k)
    with pytest.raises(TypeError):
        f(q.double(), k.double(), k.double())
    with pytest.raises(TypeError):
        f(q, k, k, k_lens=torch.ones(2, device=cuda))
    with pytest.raises(AssertionError, match="CUDA GPU required"):
        f(q.cpu(), k.cpu(), k.cpu())
