"""Causal attention over packed sequences: ``packed_attention``.

Documents of different lengths lie one behind the other along a single row
axis, and query heads may share key/value heads.  Where ``fused_attn`` is the
whole block on equal lengths, this is the attention alone, for a caller with
projections of its own.  The work is done by libmea.so through
``mea_packed_attention_forward`` and ``mea_packed_attention_backward``.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_CODES = {torch.bfloat16: _lib.MEA_BF16, torch.float16: _lib.MEA_FP16}


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` ([total, heads, N]) if the kernels can read it in place (heads' values contiguous, row and head strides
    multiples of 8 elements and at least N, 16-byte aligned), else a contiguous copy."""
    total, heads, n = t.shape
    row, head, one = t.stride()
    if (one == 1 and (total <= 1 or (row % 8 == 0 and row >= n)) and (heads == 1 or (head % 8 == 0 and head >= n))
            and t.data_ptr() % 16 == 0):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _refuse(q, k, v, cu_seqlens, scale):
    """Raises what is wrong with the arguments."""
    _lib.require_device(q.device)
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError("q, k and v must be [total, heads, N], got shapes "
                         f"{tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    total, hq, n = q.shape
    hkv = k.shape[1]
    if k.shape != v.shape or k.shape[0] != total or k.shape[2] != n:
        raise ValueError(f"k and v must be [{total}, Hkv, {n}] like q, got {tuple(k.shape)} and {tuple(v.shape)}")
    if hkv == 0 or hq == 0 or hq % hkv:
        raise ValueError(f"the query heads ({hq}) must be a positive multiple of the key/value heads ({hkv})")
    if n == 0 or n % 8 or n > 128:
        raise ValueError(f"the head dim must be a multiple of 8 up to 128, got {n}")
    if q.dtype not in _CODES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("packed_attention computes in bf16 or fp16, one type for all of q, k and v; got "
                        f"{q.dtype}, {k.dtype}, {v.dtype}")
    if cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
        raise TypeError("cu_seqlens must be a one-dimensional int32 tensor of n_seqs + 1 row numbers, got "
                        f"{cu_seqlens.dtype} of shape {tuple(cu_seqlens.shape)}")
    if not 0.0 < scale < 3e38:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    raise ValueError("all tensors must be on the same device")


def _forward(q, k, v, cu_seqlens, scale):
    """(o, what the backward needs besides q, k, v and o: their readable forms, the row log-sum-exp and the plan)."""
    dt, idx = q.dtype, q.get_device()
    if not (idx >= 0 and k.get_device() == idx and v.get_device() == idx and cu_seqlens.get_device() == idx
            and dt in _CODES and k.dtype is dt and v.dtype is dt and cu_seqlens.dtype is torch.int32
            and q.dim() == 3 and k.dim() == 3 and v.dim() == 3 and cu_seqlens.dim() == 1 and 0.0 < scale < 3e38):
        _refuse(q, k, v, cu_seqlens, scale)
    total, hq, n = q.shape
    total_k, hkv, n_k = k.shape
    n_seqs = cu_seqlens.numel() - 1
    if (k.shape != v.shape or total_k != total or n_k != n or hkv == 0 or hq == 0 or hq % hkv or n == 0 or n % 8 or n > 128
            or n_seqs < 0):
        _refuse(q, k, v, cu_seqlens, scale)
    _lib.require_index(idx)
    q, k, v = _rows(q), _rows(k), _rows(v)
    if not cu_seqlens.is_contiguous():
        cu_seqlens = cu_seqlens.contiguous()
    dims = _lib.MeaPackedDims(total, n_seqs, hq, hkv, n, _CODES[dt], scale, *q.stride()[:2], *k.stride()[:2],
                              *v.stride()[:2])
    o = q.new_empty((total, hq, n))
    if total == 0:
        return o, (q, k, v, None), dims
    L = _lib.lib()
    at = ctypes.byref(dims)
    nbytes = L.mea_packed_plan_size(at)
    # one buffer: the plan, then lse2 [total, Hq] fp32
    side = torch.empty(nbytes + 4 * total * hq, dtype=torch.uint8, device=q.device)
    p = side.data_ptr()
    _lib.launch(idx, L.mea_packed_attention_forward, at, q.data_ptr(), k.data_ptr(), v.data_ptr(), cu_seqlens.data_ptr(),
                o.data_ptr(), p + nbytes, p, nbytes, _lib.status_word(idx))
    _lib.after_launch(idx)
    return o, (q, k, v, side), dims


def _backward(ctx, grad_output):
    q, k, v, o, side = ctx.saved_tensors
    dq = q.new_empty(q.shape)
    dk = k.new_empty(k.shape)
    dv = k.new_empty(k.shape)
    if side is None:
        return dq, dk, dv, None, None
    do = _rows(grad_output)
    idx, p, L, at = q.get_device(), side.data_ptr(), _lib.lib(), ctypes.byref(ctx.dims)
    nbytes = side.numel() - 4 * q.shape[0] * q.shape[1]
    ws = torch.empty(L.mea_packed_backward_workspace_size(at), dtype=torch.uint8, device=q.device)
    _lib.launch(idx, L.mea_packed_attention_backward, at, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                do.data_ptr(), *do.stride()[:2], p + nbytes, p, nbytes, ws.data_ptr(), ws.numel(), dq.data_ptr(),
                dk.data_ptr(), dv.data_ptr(), _lib.status_word(idx))
    _lib.after_launch(idx)
    return dq, dk, dv, None, None


_backward_once = once_differentiable(_backward)


class PackedAttentionFunction(torch.autograd.Function):
    """Autograd node of ``packed_attention``.  Kept for the backward: q, k, v, o, the row log-sum-exp (fp32
    [total, Hq]) and the list of tiles that the forward made from ``cu_seqlens``."""

    @staticmethod
    def forward(ctx, q, k, v, cu_seqlens, scale):
        o, (q, k, v, side), ctx.dims = _forward(q, k, v, cu_seqlens, scale)
        ctx.save_for_backward(q, k, v, o, side)
        return o

    @staticmethod
    def backward(ctx, grad_output):
        # The gradients have no derivative of their own; the marking costs host time, so only where one could be taken.
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, grad_output)


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                     scale: float | None = None) -> torch.Tensor:
    """Causal softmax attention over packed sequences with grouped heads.

    ``q`` is [total, Hq, N], ``k`` and ``v`` are [total, Hkv, N] (bf16 or fp16, any row and head strides, so views of a
    joint projection are fine); query head h reads key/value head h // (Hq // Hkv).  ``cu_seqlens`` (int32 on the same
    device, n_seqs + 1 values) gives the rows: sequence s owns rows cu_seqlens[s] .. cu_seqlens[s+1], which may be none.
    N is a multiple of 8 up to 128.  ``scale`` multiplies the scores (default 1/sqrt(N)).

    Returns o [total, Hq, N], contiguous.  Rows that no sequence owns (before the first, behind the last) are zero in o
    and in every gradient, whatever they hold in q, k, v and the incoming gradient.  The lengths stay on the device:
    nothing is copied to the host, and a captured call follows the values that ``cu_seqlens`` has at each replay.  A
    ``cu_seqlens`` that does not rise from >= 0 to <= total gives zeros and a MeaError at a later call or at
    ``check_device_status()``.  The same call gives the same bits."""
    scale = float(q.shape[-1] ** -0.5 if scale is None else scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return PackedAttentionFunction.apply(q, k, v, cu_seqlens, scale)
    return _forward(q, k, v, cu_seqlens, scale)[0]
