"""Attention over head tensors, with autograd, on the sm_100a kernels.

``fused_attention(q, k, v, ...)`` takes the [B, S, H, D] tensors that
``fused_qk_norm_rope``, ``fused_qk_norm_mrope`` and ``apply_rope_qk`` return:
whole sequences, a chunk of new tokens over a longer cache, single tokens,
padded batches (``q_lens``, ``k_lens``) and packed documents
(``cu_seqlens``). Its backward recomputes the probabilities from the saved row
statistics. The reference has no attention of its own.
"""
from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from .._lib import address
from .fused_norm_qkv_rope import _head_strides, _heads
from .rope import _out_like


_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _addressable(t):
    """_heads, with tensors that repeat a row of memory written out (a tensor
    map cannot describe a stride of 0)."""
    if t.is_contiguous():
        return _heads(t)
    st = t.stride()
    if 0 in st and any(n > 1 and s == 0 for n, s in zip(t.shape, st)):
        t = t.contiguous()
    return _heads(t)


def _sequence_arg(x, n: int, device, name: str):
    """Lengths [n] or offsets [n] as a contiguous int32 or int64 tensor."""
    if x is None:
        return None
    if x.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"[Bloth] {name} must be int32 or int64, got {x.dtype}")
    if x.dim() != 1 or (n is not None and x.numel() != n):
        raise ValueError(f"[Bloth] {name} must have shape [{'n + 1' if n is None else n}], got "
                         f"{tuple(x.shape)}")
    if x.device != device:
        raise ValueError(f"[Bloth] {name} must be on {device}, got {x.device}")
    return x.contiguous()


def _sequences(q, k, q_lens, k_lens, cu_q, cu_k):
    """(q_seq, k_seq, packed) of the C ABI."""
    device = q.device
    batch = q.shape[0] if q.dim() == 4 else 1
    if cu_q is not None or cu_k is not None:
        if q_lens is not None or k_lens is not None:
            raise ValueError("[Bloth] give lengths (q_lens, k_lens) or offsets (cu_seqlens), "
                             "not both")
        if cu_q is None:
            raise ValueError("[Bloth] cu_seqlens_k needs cu_seqlens")
        if batch != 1:
            raise ValueError("[Bloth] packed sequences take [T, H, D] or [1, T, H, D] tensors")
        cu_q = _sequence_arg(cu_q, None, device, "cu_seqlens")
        if cu_q.numel() < 2:
            raise ValueError("[Bloth] cu_seqlens needs at least two offsets")
        if cu_k is None:
            if k.shape[-3] != q.shape[-3]:
                raise ValueError("[Bloth] q and k differ in length: give cu_seqlens_k too")
            cu_k = cu_q
        else:
            cu_k = _sequence_arg(cu_k, cu_q.numel(), device, "cu_seqlens_k")
        if cu_k.dtype != cu_q.dtype:
            cu_q, cu_k = cu_q.long(), cu_k.long()
        return cu_q, cu_k, cu_q.numel() - 1
    if q_lens is None and k_lens is None:
        return None, None, 0
    q_lens = _sequence_arg(q_lens, batch, device, "q_lens")
    k_lens = _sequence_arg(k_lens, batch, device, "k_lens")
    if q_lens is not None and k_lens is not None and q_lens.dtype != k_lens.dtype:
        q_lens, k_lens = q_lens.long(), k_lens.long()
    return q_lens, k_lens, 0


def _seq_dtype(q_seq, k_seq) -> int:
    t = q_seq if q_seq is not None else k_seq
    return _lib.I32 if t is None else _lib.dtype_code(t.dtype)


def _workspace(entry: str, device, *args):
    n = _lib.workspace_bytes(entry, device, *args)
    return (torch.empty(n, dtype=torch.uint8, device=device) if n else None), n


def _contiguous_like(t):
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def attention_forward(q4, k4, v4, q_seq, k_seq, packed, scale, causal, window, want_lse=True,
                      want_rest=False):
    """(out, lse, rest) of addressable head tensors: lse if wanted, and for
    16-bit tensors what rounding took off out, for the backward."""
    B, Sq, Hq, D = q4.shape
    Sk, Hk = k4.shape[1], k4.shape[2]
    out = _contiguous_like(q4)
    rest = torch.empty_like(out) if want_rest and q4.dtype != torch.float32 else None
    lse = q4.new_empty((B, Hq, Sq), dtype=torch.float32) if want_lse else None
    code = _lib.dtype_code(q4.dtype)
    ws, n = _workspace("bloth_attention_fwd_workspace_bytes", q4.device, B, Sq, Sk, Hq, Hk, D,
                       packed, code)
    rc = _lib.call("bloth_attention_fwd", q4, address(q4), _head_strides(q4), address(k4),
                   _head_strides(k4), address(v4), _head_strides(v4), address(out),
                   _head_strides(out), address(rest), address(lse), address(q_seq),
                   address(k_seq), _seq_dtype(q_seq, k_seq), packed, B, Sq, Sk, Hq, Hk, D, scale,
                   int(causal), window, code, address(ws), n, _lib.stream_of(q4))
    _lib.check(rc, "attention forward")
    return out, lse, rest


def attention_backward(do4, q4, k4, v4, out, rest, lse, q_seq, k_seq, packed, scale, causal, window,
                       want_q=True, want_kv=True):
    """(dq, dk, dv); None for those not wanted."""
    B, Sq, Hq, D = q4.shape
    Sk, Hk = k4.shape[1], k4.shape[2]
    dq = _out_like(q4) if want_q else None
    dk, dv = (_out_like(k4), _out_like(v4)) if want_kv else (None, None)
    code = _lib.dtype_code(q4.dtype)
    ws, n = _workspace("bloth_attention_bwd_workspace_bytes", q4.device, B, Sq, Sk, Hq, Hk, D,
                       packed, code)
    rc = _lib.call("bloth_attention_bwd", q4, address(do4), _head_strides(do4), address(q4),
                   _head_strides(q4), address(k4), _head_strides(k4), address(v4),
                   _head_strides(v4), address(out), _head_strides(out), address(rest),
                   address(lse), address(dq), _head_strides(dq), address(dk), _head_strides(dk),
                   address(dv), _head_strides(dv), address(q_seq), address(k_seq),
                   _seq_dtype(q_seq, k_seq), packed, B, Sq, Sk, Hq, Hk, D, scale, int(causal),
                   window, code, address(ws), n, _lib.stream_of(q4))
    _lib.check(rc, "attention backward")
    return dq, dk, dv


class _AttentionFunction(torch.autograd.Function):

    @staticmethod
    def forward(ctx, q, k, v, want_lse, *how):
        q4, k4, v4 = _addressable(q), _addressable(k), _addressable(v)
        out, lse, rest = attention_forward(q4, k4, v4, *how, want_rest=True)
        ctx.save_for_backward(q4, k4, v4, out, rest, lse, *how[:2])
        ctx.how = how[2:]
        if q.dim() == 3:
            out = out[0]
        if not want_lse:
            return out
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, *_):
        q4, k4, v4, out, rest, lse, q_seq, k_seq = ctx.saved_tensors
        want = ctx.needs_input_grad
        dq, dk, dv = attention_backward(_addressable(dout), q4, k4, v4, out, rest, lse, q_seq,
                                        k_seq, *ctx.how, want[0], want[1] or want[2])
        if dout.dim() == 3:
            dq, dk, dv = (None if g is None else g[0] for g in (dq, dk, dv))
        return (dq, dk if want[1] else None, dv if want[2] else None, None, None, None, None, None,
                None, None)


def fused_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool = True,
                    window: int | None = None, scale: float | None = None,
                    q_lens: torch.Tensor | None = None, k_lens: torch.Tensor | None = None,
                    cu_seqlens: torch.Tensor | None = None,
                    cu_seqlens_k: torch.Tensor | None = None, return_lse: bool = False):
    """softmax(scale * q k^T) v of q [B, Sq, Hq, D] and k, v [B, Sk, Hk, D].

    Hq is a multiple of Hk (query head h reads key head h // (Hq // Hk)); D is
    64, 128 or 256; bf16, fp16 or fp32, all three alike. ``scale`` defaults to
    1/sqrt(D). ``causal``: query i sees keys up to i + klen - qlen, so the last
    query sees the last key. ``window`` (causal only) leaves it the last
    ``window`` of those.

    ``q_lens`` and ``k_lens`` [B] (int32 or int64, on the device): the rows in
    use at the start of each batch row. ``cu_seqlens`` [n + 1]: the offsets of
    n sequences packed in [T, H, D] (or [1, T, H, D]) tensors;
    ``cu_seqlens_k`` where the keys have their own. Lengths and offsets are
    read on the device and clamped to the tensors. Rows outside of every
    sequence and rows that see no key get zeros, and no gradient; their inputs
    are never used, whatever they hold, nor are keys that no row sees. A key
    that some rows of its sequence see has to be finite for all of them (a
    probability of 0 times an infinity is not a number).

    Scores, statistics and sums are fp32. With 16-bit tensors the probabilities
    and their gradient are rounded to the tensors' type where they enter a
    product (as two terms where rows see at most 128 keys), which puts results
    of many keys about 1.4 times as far off as rounding the result alone; fp32
    tensors have none of it. For the backward of 16-bit tensors the forward
    keeps, beside q, k, v, out and lse, what rounding took off out: a second
    tensor of out's size until the backward. First derivatives in reverse mode
    only; others are refused.

    Returns out, shaped as q; with ``return_lse`` also the fp32 logarithms of
    the rows' sums of exponentials [B, Hq, Sq] ([Hq, S] for 3-D tensors), -inf
    for rows that see nothing, without a gradient.
    """
    _lib.require_cuda(q, k, v, q_lens, k_lens, cu_seqlens, cu_seqlens_k)
    shape, shape_k, dtype = q.shape, k.shape, q.dtype
    dim = len(shape)
    if dim not in (3, 4) or len(shape_k) != dim or v.dim() != dim:
        raise ValueError("[Bloth] q, k and v must be [B, S, H, D] or [S, H, D]")
    if k.dtype != dtype or v.dtype != dtype:
        raise TypeError(f"[Bloth] q, k and v differ in dtype: {dtype}, {k.dtype}, {v.dtype}")
    if dtype not in _DTYPES:
        raise TypeError(f"[Bloth] unsupported dtype {dtype}")
    if k.device != q.device or v.device != q.device:
        raise ValueError("[Bloth] q, k and v must be on one device")
    Hq, D = shape[-2:]
    Hk = shape_k[-2]
    if v.shape != shape_k or shape_k[-1] != D or (dim == 4 and shape_k[0] != shape[0]):
        raise ValueError(f"[Bloth] shapes do not match: q {tuple(shape)}, k {tuple(shape_k)}, "
                         f"v {tuple(v.shape)}")
    if D not in (64, 128, 256):
        raise ValueError(f"[Bloth] head_dim {D} is not one of 64, 128, 256")
    if Hk == 0 or Hq == 0 or Hq % Hk:
        raise ValueError(f"[Bloth] {Hq} query heads over {Hk} key heads")
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    elif not 0.0 < scale < math.inf:
        raise ValueError(f"[Bloth] scale must be positive and finite, got {scale}")
    if window is not None and (not causal or window < 1):
        raise ValueError("[Bloth] window must be at least 1, and needs causal=True")
    q_seq, k_seq, packed = _sequences(q, k, q_lens, k_lens, cu_seqlens, cu_seqlens_k)
    how = (q_seq, k_seq, packed, float(scale), bool(causal), int(window or 0))
    if (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)) or \
            _lib.has_tangent(q, k, v):
        out = _AttentionFunction.apply(q, k, v, return_lse, *how)
        if not return_lse:
            return out
        out, lse = out
    else:
        out, lse, _ = attention_forward(_addressable(q), _addressable(k), _addressable(v), *how,
                                        want_lse=return_lse)
        if dim == 3:
            out = out[0]
    if not return_lse:
        return out
    return out, lse[0] if dim == 3 else lse
