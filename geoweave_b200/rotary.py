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


@dataclass(frozen=True)
class RotaryAxes:
    """How a head's columns are divided among the axes, and the angles' tables: ``cos`` / ``sin`` fp32
    ``[positions, sum(widths) / 2]``, the axes' angles side by side.  Made once (``rotary_axes``) or filled with tables of
    the caller's own, and checked once, here."""
    widths: Tuple[int, ...]
    cos: torch.Tensor
    sin: torch.Tensor

    def __post_init__(self):
        widths = tuple(int(w) for w in self.widths)
        if not 1 <= len(widths) <= 4 or any(w <= 0 or w % 2 for w in widths):
            raise ValueError(f"widths must name one to four axes with even, positive numbers of columns, got {widths}")
        half = sum(widths) // 2
        for t in (self.cos, self.sin):
            if t.dim() != 2 or t.shape[1] != half or t.dtype != torch.float32 or t.shape != self.cos.shape or t.shape[0] < 1:
                raise ValueError(f"cos and sin must be float32 [positions, {half}]")
        object.__setattr__(self, "widths", widths)
        object.__setattr__(self, "cos", self.cos.detach().contiguous())
        object.__setattr__(self, "sin", self.sin.detach().contiguous())
        object.__setattr__(self, "_c_widths", (c_int * len(widths))(*widths))
        object.__setattr__(self, "_columns", 2 * half)


def rotary_axes(widths: Sequence[int], max_position: int, device, frequency: Union[float, Sequence[float]] = 100.0) -> RotaryAxes:
    """Tables for positions ``0 .. max_position - 1``: axis ``a`` turns its pair ``j`` by
    ``position * frequency[a] ** (-2 j / widths[a])``.  Angles and their cosines and sines are computed in 64 bits, since a
    far position's angle has lost its fraction in 32, and rounded once to fp32."""
    widths = tuple(int(w) for w in widths)
    if any(w <= 0 for w in widths):
        raise ValueError(f"widths must be positive, got {widths}")
    bases = [float(frequency)] * len(widths) if isinstance(frequency, (int, float)) else [float(f) for f in frequency]
    if len(bases) != len(widths) or any(not f > 0.0 for f in bases):
        raise ValueError("frequency must be one positive number, or one for each axis")
    if int(max_position) < 1:
        raise ValueError(f"max_position must be at least 1, got {max_position}")
    with torch.inference_mode(False):  # kept across calls: tables made during inference serve training too
        position = torch.arange(int(max_position), device=device, dtype=torch.float64)
        angles = torch.cat([position[:, None] * f ** (-torch.arange(0, w, 2, device=device, dtype=torch.float64) / w)
                            for w, f in zip(widths, bases)], 1)
        return RotaryAxes(widths, angles.cos().float().contiguous(), angles.sin().float().contiguous())


def _strides(x):
    """Element strides {batch, token, head}; a dimension of one element may carry any stride."""
    st = x.stride()
    if x.dim() == 3:
        st = (0, *st)
        return _lib.i64x3([0, st[1] if x.shape[0] > 1 else 0, st[2] if x.shape[1] > 1 else 0])
    return _lib.i64x3([st[d] if x.shape[d] > 1 else 0 for d in range(3)])


def _rotate(q, k, pos, axes: RotaryAxes, inverse: bool):
    dev = _lib.require_cuda(q, k, pos, axes.cos, axes.sin)
    shape, n_axes = q.shape, len(axes.widths)
    if len(shape) not in (3, 4):
        raise ValueError(f"q must be [N,H,D] or [B,N,H,D], got shape={tuple(shape)}")
    B, N, H, D = shape if len(shape) == 4 else (1, *shape)
    Hk = 0
    if k is not None:
        if k.dim() != len(shape) or k.shape[:-2] != shape[:-2] or k.shape[-1] != D:
            raise ValueError(f"k shape {tuple(k.shape)} does not match q {tuple(shape)} (only the number of heads may differ)")
        if k.dtype != q.dtype:
            raise TypeError("All tensors must have the same type")
        Hk = k.shape[-2]
    if axes._columns > D or D > 256:
        raise ValueError(f"the axes' widths {axes.widths} must fit a head dim of at most 256, got {D}")
    if H < 1 or (k is not None and Hk < 1):
        raise ValueError("q and k need at least one head")
    if pos.shape != shape[:-2] + (n_axes,):
        raise ValueError(f"pos must be {list(shape[:-2]) + [n_axes]}, got shape={tuple(pos.shape)}")
    if pos.dtype is not torch.int64 and pos.dtype is not torch.int32:
        raise TypeError("pos must be int64 or int32")
    code = _lib.dtype_code(q)
    pos = pos.contiguous()
    if q.stride(-1) != 1:
        q = q.contiguous()
    if k is not None and k.stride(-1) != 1:
        k = k.contiguous()
    q_out = torch.empty(shape, device=dev, dtype=q.dtype)
    k_out = None if k is None else torch.empty(k.shape, device=dev, dtype=q.dtype)
    if B == 0 or N == 0:
        return q_out, k_out
    lib = _lib.load()
    with _lib.on_device(dev):
        rc = lib.gw_rotary_axes(q.data_ptr(), _lib.ptr(k), code, B, N, H, Hk, D, _strides(q), None if k is None else _strides(k),
                                pos.data_ptr(), int(pos.dtype is torch.int64), n_axes, axes._c_widths, axes.cos.data_ptr(), axes.sin.data_ptr(),
                                axes.cos.shape[0], int(inverse), q_out.data_ptr(), _lib.ptr(k_out), _lib.status_word(dev).data_ptr(),
                                _lib.stream_ptr(dev))
    _lib.check(rc, "gw_rotary_axes")
    if _lib.debug_enabled():
        _lib.check_status(dev)
    return q_out, k_out


class _RotaryAxesFunc(torch.autograd.Function):
    """The gradient of a rotation is the rotation by the opposite angle, so nothing but positions and tables is kept."""

    @staticmethod
    def forward(ctx, q, k, pos, axes):
        ctx.axes = axes
        ctx.save_for_backward(pos, axes.cos, axes.sin)  # the tables too, so that a change in between is noticed
        return _rotate(q, k, pos, axes, False)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk):
        pos, _, _ = ctx.saved_tensors
        if all(ctx.needs_input_grad[:2]):
            return (*_rotate(dq, dk, pos, ctx.axes, True), None, None)
        if ctx.needs_input_grad[0]:
            return _rotate(dq, None, pos, ctx.axes, True)[0], None, None, None
        return None, _rotate(dk, None, pos, ctx.axes, True)[0], None, None


def apply_rotary_axes(q: torch.Tensor, k: Optional[torch.Tensor], pos: torch.Tensor, axes: RotaryAxes):
    """Turn ``q [N,H,D]`` (or ``[B,N,H,D]``) and, in the same launch, ``k`` (``None``, or the same with its own number of heads)
    by the positions ``pos`` int64 or int32 ``[N, axes]`` (or ``[B,N,axes]``); returns contiguous ``(q, k)``, differentiable in
    both.  Inputs may be slices of a fused projection's output.  A position outside the tables is reported by
    ``geoweave_b200.check_status()`` and counts as 0."""
    if _lib.wants_autograd(q) if k is None else _lib.wants_autograd(q, k):
        if k is None:
            return _RotaryQOnly.apply(q, pos, axes), None
        return _RotaryAxesFunc.apply(q, k, pos, axes)
    with torch.no_grad():
        return _rotate(q, k, pos, axes, False)


class _RotaryQOnly(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, pos, axes):
        ctx.axes = axes
        ctx.save_for_backward(pos, axes.cos, axes.sin)  # the tables too, so that a change in between is noticed
        return _rotate(q, None, pos, axes, False)[0]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq):
        pos, _, _ = ctx.saved_tensors
        return _rotate(dq, None, pos, ctx.axes, True)[0], None, None
