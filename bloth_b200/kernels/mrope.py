"""Rotary positions with several axes (time, height, width), with autograd.

Images and video give each token a position per axis; every frequency of the
rotation belongs to one axis. ``mrope_axes`` lays the axes over the
frequencies as HuggingFace's vision-language models do, and
``fused_qk_norm_mrope`` / ``apply_mrope_qk`` are ``fused_qk_norm_rope`` /
``apply_rope_qk`` with such positions: the same kernels, the same layouts, the
same gradients. The reference rotates by one position per token.
"""
from __future__ import annotations

import ctypes
from functools import lru_cache

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from .._lib import address
from .fused_norm_qkv_rope import _head_strides, _heads
from .rope import _out_like

MAX_AXES = 4


def _contiguous_like(t):
    return torch.empty_like(t, memory_format=torch.contiguous_format)


@lru_cache(maxsize=64)
def _mrope_axes(sections: tuple, interleaved: bool) -> tuple:
    if not 1 <= len(sections) <= MAX_AXES or any(n < 0 for n in sections):
        raise ValueError(f"[Bloth] sections must be 1 to {MAX_AXES} counts, got {sections}")
    n = len(sections)
    if not interleaved:
        return tuple(a for a, c in enumerate(sections) for _ in range(c))
    axes = [i % n if i % n and i // n < sections[i % n] else 0 for i in range(sum(sections))]
    if any(axes.count(a) != c for a, c in enumerate(sections)):
        raise ValueError(f"[Bloth] sections {sections} cannot be interleaved: the first axis has "
                         "too few frequencies to take turns with the others")
    return tuple(axes)


def mrope_axes(sections, interleaved: bool = False) -> tuple:
    """The axis of each of the D/2 frequencies, from the number of frequencies
    per axis (HF's ``mrope_section``; their sum is D/2). By default the axes
    follow one another. ``interleaved`` (HF's ``mrope_interleaved``): the axes take
    turns, frequency i going to axis i mod n while that axis has some left,
    and to the first axis otherwise."""
    return _mrope_axes(tuple(int(n) for n in sections), bool(interleaved))


@lru_cache(maxsize=64)
def _axes_array(axes: tuple, half: int, n: int):
    if len(axes) != half:
        raise ValueError(f"[Bloth] axes must name one axis for each of the {half} frequencies, "
                         f"got {len(axes)}")
    if any(not 0 <= a < n for a in axes):
        raise ValueError(f"[Bloth] axes must be in [0, {n}), the axes of position_ids")
    return (ctypes.c_uint8 * half)(*axes)


def _axis_positions(position_ids, B: int, S: int):
    """(positions [A, B|1, S], strides[3] axis, batch, sequence)."""
    p = position_ids
    if p.dtype not in (torch.int32, torch.int64):
        p = p.long()
    if p.dim() == 2:
        p = p.unsqueeze(1)
    if p.dim() != 3 or p.shape[2] != S or p.shape[1] not in (1, B) or \
            not 1 <= p.shape[0] <= MAX_AXES:
        raise ValueError(f"[Bloth] position_ids shape {tuple(position_ids.shape)} is not [axes, "
                         f"batch {B}, seq {S}] (or [axes, seq]) with 1 to {MAX_AXES} axes")
    return p, _lib.strides((p.stride(0), 0 if p.shape[1] == 1 else p.stride(1), p.stride(2)))


def _same_device(t, device, name: str):
    if t.device != device:
        raise ValueError(f"[Bloth] {name} must be on {device}, got {t.device}")


def _source(x4, position_ids, inv_freq, axes):
    """(positions, strides, axes array, inv_freq) of a call on x4."""
    B, S, _, D = x4.shape
    if position_ids is None or inv_freq is None:
        raise ValueError("[Bloth] position_ids and inv_freq are required")
    _same_device(position_ids, x4.device, "position_ids")
    _same_device(inv_freq, x4.device, "inv_freq")
    pos, pos_st = _axis_positions(position_ids, B, S)
    if inv_freq.dtype != torch.float32 or not inv_freq.is_contiguous():
        inv_freq = inv_freq.to(torch.float32).contiguous()
    if inv_freq.numel() != D // 2:
        raise ValueError(f"[Bloth] inv_freq must have head_dim/2 = {D // 2} elements")
    return pos, pos_st, _axes_array(tuple(axes), D // 2, pos.shape[0]), inv_freq


def _check_pair(q4, k4):
    if k4 is not None and (k4.shape[:2] != q4.shape[:2] or k4.shape[3] != q4.shape[3]):
        raise ValueError("[Bloth] q and k must share batch, sequence and head_dim")
    if k4 is not None and k4.dtype != q4.dtype:
        raise TypeError(f"[Bloth] q and k differ in dtype: {q4.dtype}, {k4.dtype}")
    if k4 is not None:
        _same_device(k4, q4.device, "k")


def _needs_grad(inv_freq, *tensors) -> bool:
    grad = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)
    return grad or _lib.has_tangent(inv_freq, *tensors)


def _weight(w, D: int, dtype, device):
    _same_device(w, device, "wq and wk")
    if w.numel() != D or w.dtype != dtype:
        raise ValueError(f"[Bloth] wq and wk must have head_dim = {D} elements of one dtype")
    return _lib.aligned16(w.contiguous())


def _norm_mrope_call(q, k, wq, wk, position_ids, inv_freq, axes, eps, weight_offset, rope_scale):
    """Forward: (q_out, k_out, what the backward needs)."""
    q4, k4 = _heads(q), _heads(k)
    _check_pair(q4, k4)
    B, S, Hq, D = q4.shape
    Hk = 0 if k4 is None else k4.shape[2]
    pos, pos_st, ax, inv_freq = _source(q4, position_ids, inv_freq, axes)
    if k4 is not None and wk is None:
        raise ValueError("[Bloth] wk is required with k")
    wk = None if wk is None else _weight(wk, D, wq.dtype, q4.device)
    wq = _weight(wq, D, wq.dtype, q4.device)
    qo = _contiguous_like(q4)
    ko = None if k4 is None else _contiguous_like(k4)
    rq = q4.new_empty((B, S, Hq), dtype=torch.float32)
    rk = None if k4 is None else q4.new_empty((B, S, Hk), dtype=torch.float32)
    rc = _lib.call(
        "bloth_qk_norm_mrope_fwd", q4, address(q4), _head_strides(q4), address(k4),
        _head_strides(k4), address(wq), address(wk), weight_offset, address(qo),
        _head_strides(qo), address(ko), _head_strides(ko), address(rq), address(rk),
        address(pos), pos_st, _lib.dtype_code(pos.dtype), pos.shape[0], ax, address(inv_freq),
        rope_scale, B, S, Hq, Hk, D, eps, _lib.dtype_code(q4.dtype), _lib.dtype_code(wq.dtype),
        _lib.stream_of(q4))
    _lib.check(rc, "qk norm+mrope forward")
    saved = (q4, k4, wq, wk, rq, rk, pos, inv_freq), (pos_st, ax, q.dim() == 3, weight_offset,
                                                      rope_scale)
    if q.dim() == 3:
        qo, ko = qo[0], None if ko is None else ko[0]
    return qo, ko, saved


class _QKNormMRoPEFunction(torch.autograd.Function):

    @staticmethod
    def forward(ctx, *args):
        qo, ko, (tensors, ctx.meta) = _norm_mrope_call(*args)
        ctx.save_for_backward(*tensors)
        return qo if ko is None else (qo, ko)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        q4, k4, wq, wk, rq, rk, pos, inv_freq = ctx.saved_tensors
        pos_st, ax, flat, weight_offset, rope_scale = ctx.meta
        B, S, Hq, D = q4.shape
        Hk = 0 if k4 is None else k4.shape[2]
        gq = _heads(grads[0])
        gk = None if k4 is None else _heads(grads[1])
        dq = _contiguous_like(q4)
        dk = None if k4 is None else _contiguous_like(k4)
        dwq = torch.empty_like(wq)
        dwk = None if k4 is None else torch.empty_like(wk)
        code = _lib.dtype_code(q4.dtype)
        n = _lib.workspace_bytes("bloth_qk_norm_mrope_bwd_workspace_bytes", q4.device, B, S, D,
                                 code)
        ws = torch.empty(max(n, 1), dtype=torch.uint8, device=q4.device)
        rc = _lib.call(
            "bloth_qk_norm_mrope_bwd", q4, address(gq), _head_strides(gq), address(gk),
            _head_strides(gk), address(q4), _head_strides(q4), address(k4), _head_strides(k4),
            address(wq), address(wk), weight_offset, address(rq), address(rk), address(dq),
            _head_strides(dq), address(dk), _head_strides(dk), address(dwq), address(dwk),
            address(pos), pos_st, _lib.dtype_code(pos.dtype), pos.shape[0], ax,
            address(inv_freq), rope_scale, B, S, Hq, Hk, D, code, _lib.dtype_code(wq.dtype),
            address(ws), n, _lib.stream_of(q4))
        _lib.check(rc, "qk norm+mrope backward")
        if flat:
            dq, dk = dq[0], None if dk is None else dk[0]
        return dq, dk, dwq, dwk, None, None, None, None, None, None


def _mrope_launch(q4, qo, k4, ko, pos, pos_st, ax, inv_freq, scale, transpose):
    B, S, Hq, D = q4.shape
    rc = _lib.call("bloth_mrope", q4, address(q4), _head_strides(q4), address(qo),
                   _head_strides(qo), address(k4), _head_strides(k4), address(ko),
                   _head_strides(ko), address(pos), pos_st, _lib.dtype_code(pos.dtype),
                   pos.shape[0], ax, address(inv_freq), scale, B, S, Hq,
                   0 if k4 is None else k4.shape[2], D, int(transpose),
                   _lib.dtype_code(q4.dtype), _lib.stream_of(q4))
    _lib.check(rc, "mrope")


def _mrope_call(q, k, position_ids, inv_freq, axes, scale):
    """Forward: (q_out, k_out, what the backward needs)."""
    q4, k4 = _heads(q), _heads(k)
    _check_pair(q4, k4)
    pos, pos_st, ax, inv_freq = _source(q4, position_ids, inv_freq, axes)
    qo = _out_like(q4)
    ko = None if k4 is None else _out_like(k4)
    _mrope_launch(q4, qo, k4, ko, pos, pos_st, ax, inv_freq, scale, False)
    saved = (pos, inv_freq), (pos_st, ax, scale, q.dim() == 3, k4 is not None)
    if q.dim() == 3:
        qo, ko = qo[0], None if ko is None else ko[0]
    return qo, ko, saved


class _MRoPEFunction(torch.autograd.Function):

    @staticmethod
    def forward(ctx, *args):
        qo, ko, (tensors, ctx.meta) = _mrope_call(*args)
        ctx.save_for_backward(*tensors)
        return qo if ko is None else (qo, ko)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        pos, inv_freq = ctx.saved_tensors
        pos_st, ax, scale, flat, has_k = ctx.meta
        gq = _heads(grads[0])
        gk = _heads(grads[1]) if has_k else None
        dq, dk = _out_like(gq), None if gk is None else _out_like(gk)
        _mrope_launch(gq, dq, gk, dk, pos, pos_st, ax, inv_freq, scale, True)
        if flat:
            dq, dk = dq[0], None if dk is None else dk[0]
        return dq, dk, None, None, None, None


def fused_qk_norm_mrope(q: torch.Tensor, k: torch.Tensor | None, wq: torch.Tensor,
                        wk: torch.Tensor | None, position_ids: torch.Tensor,
                        inv_freq: torch.Tensor, axes, eps: float = 1e-6,
                        weight_offset: float = 0.0, rope_scale: float = 1.0):
    """Per-head RMSNorm + rotate-half RoPE of q [B, S, Hq, D] and k [B, S, Hk, D]
    by positions of several axes.

    ``position_ids`` [A, B, S], [A, 1, S] or [A, S], A from 1 to 4; ``axes``
    the axis of each of the D/2 frequencies (:func:`mrope_axes`): pair
    (d, d + D/2) turns by float32(position of axis axes[d]) * inv_freq[d].
    The rest is :func:`fused_qk_norm_rope`'s: weight gradients for both norms,
    ``weight_offset``, ``rope_scale``, k may be None. Returns (q_out, k_out),
    or q_out alone."""
    _lib.require_cuda(q, k, wq, wk, position_ids, inv_freq)
    args = (q, k, wq, wk, position_ids, inv_freq, axes, float(eps), float(weight_offset),
            float(rope_scale))
    if _needs_grad(inv_freq, q, k, wq, wk):
        return _QKNormMRoPEFunction.apply(*args)
    qo, ko, _ = _norm_mrope_call(*args)
    return qo if ko is None else (qo, ko)


def apply_mrope_qk(q: torch.Tensor, k: torch.Tensor | None, position_ids: torch.Tensor,
                   inv_freq: torch.Tensor, axes, rope_scale: float = 1.0):
    """Rotate-half RoPE of q [B, S, Hq, D] and k [B, S, Hk, D] (or q alone, k
    None) by positions of several axes, in one launch; see
    :func:`fused_qk_norm_mrope`."""
    _lib.require_cuda(q, k, position_ids, inv_freq)
    args = (q, k, position_ids, inv_freq, axes, float(rope_scale))
    if _needs_grad(inv_freq, q, k):
        return _MRoPEFunction.apply(*args)
    qo, ko, _ = _mrope_call(*args)
    return qo if ko is None else (qo, ko)
