"""Rotary positions with several axes (time, height, width) as an operator of its own, with its gradient.

The sparse layers turn q and k inside the fused projection (``front_end``, two axes, head dim 64).  The dense blocks around
them take q and k from other projections, need a time axis for video, other head dims, and gradients; this is the step
between such a projection and ``custom_flash_attn``.  The two-axis form with equal widths is the reference's
``RotaryPositionEmbedding2D`` (``easyvolcap/official_vggt/layers/rope.py:134-188``).
"""
from __future__ import annotations

from ctypes import c_int
from dataclasses import dataclass
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _lib

__all__ = ["RotaryAxes", "rotary_axes", "apply_rotary_axes"]


@dataclass
class RotaryAxes:
    """How a head's columns are divided among the axes, and the angles' tables: ``cos`` / ``sin`` fp32
    ``[positions, sum(widths) / 2]``, the axes' angles side by side.  Made once (``rotary_axes``) or filled with tables of
    the caller's own."""
    widths: Tuple[int, ...]
    cos: torch.Tensor
    sin: torch.Tensor


def _checked_widths(widths) -> Tuple[int, ...]:
    widths = tuple(int(w) for w in widths)
    if not 1 <= len(widths) <= 4 or any(w <= 0 or w % 2 for w in widths):
        raise ValueError(f"widths must name one to four axes with even, positive numbers of columns, got {widths}")
    return widths


def rotary_axes(widths: Sequence[int], max_position: int, device, frequency: Union[float, Sequence[float]] = 100.0) -> RotaryAxes:
    """Tables for positions ``0 .. max_position - 1``: axis ``a`` turns its pair ``j`` by
    ``position * frequency[a] ** (-2 j / widths[a])``.  Angles and their cosines and sines are computed in 64 bits, since a
    far position's angle has lost its fraction in 32, and rounded once to fp32."""
    widths = _checked_widths(widths)
    bases = [float(frequency)] * len(widths) if isinstance(frequency, (int, float)) else [float(f) for f in frequency]
    if len(bases) != len(widths) or any(not f > 0.0 for f in bases):
        raise ValueError("frequency must be one positive number, or one for each axis")
    if int(max_position) < 1:
        raise ValueError(f"max_position must be at least 1, got {max_position}")
    position = torch.arange(int(max_position), device=device, dtype=torch.float64)
    angles = torch.cat([position[:, None] * f ** (-torch.arange(0, w, 2, device=device, dtype=torch.float64) / w)
                        for w, f in zip(widths, bases)], 1)
    return RotaryAxes(widths, angles.cos().float().contiguous(), angles.sin().float().contiguous())


def _rotate(q, k, pos, axes: RotaryAxes, inverse: bool):
    lib = _lib.load()
    dev = _lib.require_cuda(q, k, pos, axes.cos, axes.sin)
    widths = _checked_widths(axes.widths)
    if q.dim() not in (3, 4):
        raise ValueError(f"q must be [N,H,D] or [B,N,H,D], got shape={tuple(q.shape)}")
    D = q.shape[-1]
    if k is not None and (k.dim() != q.dim() or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != D):
        raise ValueError(f"k shape {tuple(k.shape)} does not match q {tuple(q.shape)} (only the number of heads may differ)")
    if k is not None and k.dtype != q.dtype:
        raise TypeError("All tensors must have the same type")
    if sum(widths) > D or D > 256:
        raise ValueError(f"the axes' widths {widths} must fit a head dim of at most 256, got {D}")
    if q.shape[-2] < 1 or (k is not None and k.shape[-2] < 1):
        raise ValueError("q and k need at least one head")
    if tuple(pos.shape) != tuple(q.shape[:-2]) + (len(widths),):
        raise ValueError(f"pos must be {list(q.shape[:-2]) + [len(widths)]}, got shape={tuple(pos.shape)}")
    if pos.dtype not in (torch.int64, torch.int32):
        raise TypeError("pos must be int64 or int32")
    half = sum(widths) // 2
    for t in (axes.cos, axes.sin):
        if t.dim() != 2 or t.shape[1] != half or t.dtype != torch.float32 or t.shape != axes.cos.shape or t.shape[0] < 1:
            raise ValueError(f"cos and sin must be float32 [positions, {half}]")
    cos, sin, pos = axes.cos.contiguous(), axes.sin.contiguous(), pos.contiguous()
    q, k = [x if x is None or x.stride(-1) == 1 or D == 1 else x.contiguous() for x in (q, k)]
    q4, k4 = [x if x is None or x.dim() == 4 else x.unsqueeze(0) for x in (q, k)]
    B, N, H, _ = q4.shape
    Hk = 0 if k is None else k4.shape[2]
    q_out = torch.empty(q.shape, device=dev, dtype=q.dtype)
    k_out = None if k is None else torch.empty(k.shape, device=dev, dtype=q.dtype)
    if B == 0 or N == 0:
        return q_out, k_out

    def strides(x):  # a dimension of one element may carry any stride
        return _lib.i64x3([x.stride(d) if x.shape[d] > 1 else 0 for d in range(3)])

    with _lib.on_device(dev):
        rc = lib.gw_rotary_axes(q4.data_ptr(), _lib.ptr(k4), _lib.dtype_code(q), B, N, H, Hk, D, strides(q4),
                                None if k is None else strides(k4), pos.data_ptr(), int(pos.dtype == torch.int64), len(widths),
                                (c_int * len(widths))(*widths), cos.data_ptr(), sin.data_ptr(), cos.shape[0], int(inverse),
                                q_out.data_ptr(), _lib.ptr(k_out), _lib.status_word(dev).data_ptr(), _lib.stream_ptr(dev))
    _lib.check(rc, "gw_rotary_axes")
    if _lib.debug_enabled():
        _lib.check_status(dev)
    return q_out, k_out


class _RotaryAxesFunc(torch.autograd.Function):
    """The gradient of a rotation is the rotation by the opposite angle, so nothing but positions and tables is kept."""

    @staticmethod
    def forward(ctx, q, k, pos, axes):
        ctx.axes = axes
        ctx.save_for_backward(pos, axes.cos, axes.sin)
        return _rotate(q, k, pos, axes, False)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk):
        pos, cos, sin = ctx.saved_tensors
        dq, dk = _rotate(dq, dk, pos, RotaryAxes(ctx.axes.widths, cos, sin), True)
        return dq, dk, None, None


def apply_rotary_axes(q: torch.Tensor, k: Optional[torch.Tensor], pos: torch.Tensor, axes: RotaryAxes):
    """Turn ``q [N,H,D]`` (or ``[B,N,H,D]``) and, in the same launch, ``k`` (``None``, or the same with its own number of heads)
    by the positions ``pos`` int64 or int32 ``[N, axes]`` (or ``[B,N,axes]``); returns contiguous ``(q, k)``, differentiable in
    both.  Inputs may be slices of a fused projection's output.  A position outside the tables is reported by
    ``geoweave_b200.check_status()`` and counts as 0."""
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        if k is None:
            return _RotaryQOnly.apply(q, pos, axes), None
        return _RotaryAxesFunc.apply(q, k, pos, axes)
    with torch.no_grad():
        return _rotate(q, k, pos, axes, False)


class _RotaryQOnly(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, pos, axes):
        ctx.axes = axes
        ctx.save_for_backward(pos, axes.cos, axes.sin)
        return _rotate(q, None, pos, axes, False)[0]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq):
        pos, cos, sin = ctx.saved_tensors
        return _rotate(dq, None, pos, RotaryAxes(ctx.axes.widths, cos, sin), True)[0], None, None
