"""Attention over packed sequences: softmax over every allowed key, forward and backward.

The dense counterpart of the sparse-index attention beside it, for the blocks around the sparse layers: frame blocks
(every view attends to itself), dense global layers (the scene is one sequence), ragged causal prompts, and single query
tokens against long key sequences.  Sequences lie back to back in ``[tokens, heads, head_dim]`` tensors and int32 border
arrays say where each begins, as the name of the kernel's entry point ``gw_packed_attn_fwd`` suggests.

The border arrays are never read on the host, so calls enqueue without synchronising and can be captured into CUDA graphs;
borders that make no sense are reported by ``geoweave_b200.check_status()``.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from .. import _lib

__all__ = ["packed_flash_attn_func", "packed_flash_attn_inference_func", "packed_attention_forward", "packed_attention_backward"]


def _scale(softmax_scale, D):
    if softmax_scale is None:
        return 1.0 / math.sqrt(D)
    scale = float(softmax_scale)
    if not 2.0 ** -126 <= scale <= 2.0 ** 127:  # as fp32, and times log2 e
        raise ValueError(f"softmax_scale must be positive and finite in fp32, at least 2**-126 and at most 2**127, got {softmax_scale}")
    return scale


def _prepared(x):
    """``x`` as the kernels can copy it in 16-byte pieces -- contiguous head dim, base and strides on 16-byte boundaries, no
    broadcast dims; a copy if it is not -- and its element strides {token, head}."""
    T, H, D = x.shape
    if not x.is_contiguous():
        st, es = x.stride(), x.element_size()
        # a dimension of one element may carry any stride, so it gets that of a contiguous tensor
        token, head = st[0] if T > 1 else H * D, st[1] if H > 1 else D
        if st[2] == 1 and x.data_ptr() % 16 == 0 and token > 0 and head > 0 and token * es % 16 == 0 and head * es % 16 == 0:
            return x, _lib.i64x2((token, head))
        x = x.contiguous()
    if x.data_ptr() % 16 != 0:  # a contiguous tensor may still start off a 16-byte boundary
        x = x.clone(memory_format=torch.contiguous_format)
    return x, _lib.i64x2((H * D, D))


def _borders(cu, name, dev):
    if cu.dim() != 1 or cu.numel() < 1:
        raise ValueError(f"{name} must be one-dimensional with one more entry than there are sequences, got shape={tuple(cu.shape)}")
    if cu.dtype != torch.int32:
        raise TypeError(f"{name} must be int32")
    if cu.device != dev:
        raise ValueError("all tensors must be on the same CUDA device")
    return cu.contiguous()


def _checked(q, k, v, cu_seqlens_q, cu_seqlens_k):
    dev = _lib.require_cuda(q, k, v, cu_seqlens_q, cu_seqlens_k)
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError("q, k, v must be [tokens, heads, head_dim]")
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError("All tensors must have the same type")
    _lib.dtype_code(q)
    T, H, D = q.shape
    S, Hk = k.shape[:2]
    if k.shape[2] != D or v.shape != k.shape:
        raise ValueError(f"k/v shape {tuple(k.shape)}/{tuple(v.shape)} does not match q {tuple(q.shape)}")
    if H < 1 or Hk < 1 or H % Hk != 0:
        raise ValueError(f"the number of query heads ({H}) must be a multiple of the number of key heads ({Hk})")
    if D < 1 or D > 128 or D % 8 != 0:
        raise ValueError(f"head dimensions up to 128 that are a multiple of 8 are supported, got {D}")
    if H > 65535 or max(T, S) > 0x7fffff00:
        raise ValueError("at most 65535 heads and 2**31 - 256 tokens are supported")
    cu_q = _borders(cu_seqlens_q, "cu_seqlens_q", dev)
    cu_k = cu_q if cu_seqlens_k is None else _borders(cu_seqlens_k, "cu_seqlens_k", dev)
    if cu_seqlens_k is None and T != S:
        raise ValueError("without cu_seqlens_k the keys are the queries' own tokens: q and k must have the same length")
    if cu_q.numel() != cu_k.numel():
        raise ValueError(f"cu_seqlens_q and cu_seqlens_k name different numbers of sequences ({cu_q.numel() - 1} and {cu_k.numel() - 1})")
    return dev, T, S, H, Hk, D, cu_q, cu_k


def packed_attention_forward(q, k, v, cu_seqlens_q, cu_seqlens_k=None, causal=False, softmax_scale=None, max_seqlen_q=None,
                             return_lse=False, o_low: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Shared implementation: ``(o [tokens, heads, head_dim], lse fp32 [heads, tokens] or None)``.  ``o_low``, contiguous and like
    ``o``, receives what rounding ``o`` to 16 bits took off (the backward pass wants it; not used for fp32)."""
    scale = _scale(softmax_scale, q.shape[-1])
    if max_seqlen_q is not None and int(max_seqlen_q) < 0:
        raise ValueError(f"max_seqlen_q must not be negative, got {max_seqlen_q}")
    dev, T, S, H, Hk, D, cu_q, cu_k = _checked(q, k, v, cu_seqlens_q, cu_seqlens_k)
    if o_low is not None and (o_low.shape != q.shape or o_low.dtype != q.dtype or o_low.device != dev or not o_low.is_contiguous()):
        raise ValueError("o_low must be a contiguous tensor like o")
    o = torch.empty((T, H, D), device=dev, dtype=q.dtype)
    lse = torch.empty((H, T), device=dev, dtype=torch.float32) if return_lse else None
    if T == 0:
        return o, lse
    if S == 0:
        if lse is not None:
            lse.fill_(float("-inf"))
        if o_low is not None:
            o_low.zero_()
        return o.zero_(), lse
    (q, qs), (k, ks), (v, vs) = _prepared(q), _prepared(k), _prepared(v)
    nseq, code = cu_q.shape[0] - 1, _lib.dtype_code(q)
    most = T if max_seqlen_q is None else min(T, int(max_seqlen_q))
    lib = _lib.load()
    with _lib.on_device(dev):
        nbytes = lib.gw_packed_attn_fwd_workspace_bytes(code, nseq, T, S, H, Hk, D, most)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        rc = lib.gw_packed_attn_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), code, cu_q.data_ptr(), cu_k.data_ptr(), nseq, T, S, H, Hk, D,
                                    qs, ks, vs, scale, int(bool(causal)), most, o.data_ptr(), _lib.ptr(o_low), _lib.ptr(lse),
                                    _lib.ptr(ws), nbytes, _lib.status_word(dev).data_ptr(), _lib.stream_ptr(dev))
    _lib.check(rc, "gw_packed_attn_fwd")
    if _lib.debug_enabled():
        _lib.check_status(dev)
    return o, lse


def packed_attention_backward(q, k, v, cu_seqlens_q, cu_seqlens_k, o, lse, d_out, causal=False, softmax_scale=None, o_low=None,
                              key_grads=True):
    """Gradients ``(dq, dk, dv)`` of the forward, contiguous and of the inputs' dtype.  The sums run in a fixed order
    (one kernel owns query rows, another key rows; no atomics), so results are reproducible.  ``key_grads=False``: ``(dq, None,
    None)``, and the second kernel does not run; the first always does, for the second needs its row sums."""
    scale = _scale(softmax_scale, q.shape[-1])
    dev, T, S, H, Hk, D, cu_q, cu_k = _checked(q, k, v, cu_seqlens_q, cu_seqlens_k)
    _lib.require_cuda(q, o, lse, d_out)
    if tuple(o.shape) != (T, H, D) or tuple(d_out.shape) != (T, H, D) or tuple(lse.shape) != (H, T):
        raise ValueError("o, d_out and lse must be the forward's: [tokens, heads, head_dim] twice and [heads, tokens]")
    if lse.dtype != torch.float32 or o.dtype != q.dtype:
        raise TypeError("o must have q's type and lse must be float32")
    dq = torch.empty((T, H, D), device=dev, dtype=q.dtype)
    dk, dv = [torch.empty((S, Hk, D), device=dev, dtype=q.dtype) if key_grads else None for _ in range(2)]
    if T == 0 or S == 0:
        return tuple(x if x is None else x.zero_() for x in (dq, dk, dv))
    (q, qs), (k, ks), (v, vs), (d_out, ds) = _prepared(q), _prepared(k), _prepared(v), _prepared(d_out.to(q.dtype))
    o, lse = _prepared(o.contiguous())[0], lse.contiguous()
    if o_low is not None and (o_low.shape != o.shape or o_low.dtype != o.dtype or o_low.device != dev or not o_low.is_contiguous()):
        raise ValueError("o_low must be the forward's")
    nseq = cu_q.numel() - 1
    lib = _lib.load()
    nbytes = lib.gw_packed_attn_bwd_workspace_bytes(T, H)
    with _lib.on_device(dev):
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        rc = lib.gw_packed_attn_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), _lib.ptr(o_low), lse.data_ptr(), d_out.data_ptr(),
                                    _lib.dtype_code(q), cu_q.data_ptr(), cu_k.data_ptr(), nseq, T, S, H, Hk, D, qs, ks, vs, ds,
                                    scale, int(bool(causal)), dq.data_ptr(), _lib.ptr(dk), _lib.ptr(dv), ws.data_ptr(), nbytes,
                                    _lib.status_word(dev).data_ptr(), _lib.stream_ptr(dev))
    _lib.check(rc, "gw_packed_attn_bwd")
    if _lib.debug_enabled():
        _lib.check_status(dev)
    return dq, dk, dv


class _PackedFlashAttn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_seqlens_q, cu_seqlens_k, causal, softmax_scale, max_seqlen_q):
        o_low = None if q.dtype is torch.float32 else torch.empty(q.shape, device=q.device, dtype=q.dtype)
        o, lse = packed_attention_forward(q, k, v, cu_seqlens_q, cu_seqlens_k, causal, softmax_scale, max_seqlen_q, True, o_low)
        ctx.save_for_backward(q, k, v, cu_seqlens_q, cu_seqlens_k, o, lse, o_low)
        ctx.causal, ctx.softmax_scale = causal, softmax_scale
        return o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out):
        q, k, v, cu_q, cu_k, o, lse, o_low = ctx.saved_tensors
        dq, dk, dv = packed_attention_backward(q, k, v, cu_q, cu_k, o, lse, d_out, ctx.causal, ctx.softmax_scale, o_low,
                                               any(ctx.needs_input_grad[1:3]))
        return dq, dk, dv, None, None, None, None, None


def packed_flash_attn_func(q, k, v, cu_seqlens_q, cu_seqlens_k=None, causal: bool = False, softmax_scale: Optional[float] = None,
                           max_seqlen_q: Optional[int] = None) -> torch.Tensor:
    """Attention of packed sequences, differentiable in q, k and v.

    ``q [total_q, H, D]``, ``k, v [total_k, Hk, D]`` (bf16 / fp16 / fp32, ``D`` a multiple of 8 up to 128, ``H`` a multiple of
    ``Hk``: query head ``h`` reads key head ``h // (H // Hk)``).  ``cu_seqlens_q``, ``cu_seqlens_k`` int32 ``[sequences + 1]``
    on the same device: sequence ``b`` holds rows ``cu[b]`` to ``cu[b + 1]``; ``cu_seqlens_k=None`` means the queries' own
    tokens.  ``causal``: the last query of a sequence sees all its keys, the one before it one key less, and so on.
    ``max_seqlen_q``: an upper bound on the queries of one sequence, if the caller knows one.  Up to 16 query rows a key head
    (queries times heads of a group) the work is then divided along the keys; without the bound such a batch takes the kernel for prompts, where each
    query head reads all keys for a tile of rows that is almost empty: give it for single new tokens (24 of them against 129 to 33 312 keys each: 38 us, and 309 without).
    A bound that is too small sets the status word and leaves rows unwritten.

    Under autograd a 16-bit call keeps, beside its output, a second tensor of that size until the backward pass: what rounding the output took
    off, for exact row sums.  Without gradients (``packed_flash_attn_inference_func``) there is none.  Derivatives are first-order and
    backward only: forward-mode tangents and second derivatives are refused.

    Rows without an allowed key and rows behind the last sequence give zeros (gradients too).  Non-finite values of ``k`` and
    ``v`` stay within their own sequence; within a causal sequence they may also reach rows before them.
    """
    if _lib.wants_autograd(q, k, v):
        return _PackedFlashAttn.apply(q, k, v, cu_seqlens_q, cu_seqlens_k, bool(causal), softmax_scale, max_seqlen_q)
    with torch.no_grad():
        return packed_attention_forward(q, k, v, cu_seqlens_q, cu_seqlens_k, causal, softmax_scale, max_seqlen_q)[0]


def packed_flash_attn_inference_func(q, k, v, cu_seqlens_q, cu_seqlens_k=None, causal: bool = False,
                                     softmax_scale: Optional[float] = None, max_seqlen_q: Optional[int] = None,
                                     return_lse: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """As ``packed_flash_attn_func`` without gradients: ``(o, lse | None)``, ``lse`` fp32 ``[H, total_q]`` (natural logarithm,
    ``-inf`` for rows without an allowed key)."""
    with torch.no_grad():
        return packed_attention_forward(q, k, v, cu_seqlens_q, cu_seqlens_k, causal, softmax_scale, max_seqlen_q, return_lse)
