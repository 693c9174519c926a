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


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` ([total, heads, N]) if the kernels can read it in place (heads' values contiguous, row and head strides
    multiples of 8 elements and at least N, 16-byte aligned), else a contiguous copy."""
    total, heads, n = t.shape
    row, head, one = t.stride()
    if (one == 1 and (total <= 1 or (row % 8 == 0 and row >= n)) and (heads == 1 or (head % 8 == 0 and head >= n))
            and t.data_ptr() % 16 == 0):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _check(q, k, v, cu_seqlens, scale):
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
    if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("packed_attention computes in bf16 or fp16, one type for all of q, k and v; got "
                        f"{q.dtype}, {k.dtype}, {v.dtype}")
    if cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
        raise TypeError("cu_seqlens must be a one-dimensional int32 tensor of n_seqs + 1 row numbers, got "
                        f"{cu_seqlens.dtype} of shape {tuple(cu_seqlens.shape)}")
    if k.device != q.device or v.device != q.device or cu_seqlens.device != q.device:
        raise ValueError("all tensors must be on the same device")
    if not 0.0 < scale < 3e38:
        raise ValueError(f"scale must be positive and finite, got {scale}")


class PackedAttentionFunction(torch.autograd.Function):
    """Autograd node of ``packed_attention``.  Kept for the backward: q, k, v, o, the row log-sum-exp (fp32
    [total, Hq]) and the list of tiles that the forward made from ``cu_seqlens``."""

    @staticmethod
    def forward(ctx, q, k, v, cu_seqlens, scale):
        _check(q, k, v, cu_seqlens, scale)
        q, k, v, cu_seqlens = _rows(q), _rows(k), _rows(v), cu_seqlens.contiguous()
        total, hq, n = q.shape
        dims = _lib.MeaPackedDims(total, cu_seqlens.numel() - 1, hq, k.shape[1], n, _lib.DTYPE_CODES[q.dtype], scale,
                                  q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1))
        o = torch.empty(total, hq, n, dtype=q.dtype, device=q.device)
        if total == 0:
            lse = plan = None
        else:
            with _lib.on_device(q.device):
                _lib.poll_status_eager(q.device)
                L = _lib.lib()
                nbytes = L.mea_packed_plan_size(ctypes.byref(dims))
                lse = torch.empty(total, hq, dtype=torch.float32, device=q.device)
                plan = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
                _lib.check(L.mea_packed_attention_forward(
                    ctypes.byref(dims), q.data_ptr(), k.data_ptr(), v.data_ptr(), cu_seqlens.data_ptr(), o.data_ptr(),
                    lse.data_ptr(), plan.data_ptr(), nbytes, _lib.status_word(q.device),
                    _lib.stream_ptr(q.device)))
                _lib.note_status_eager(q.device)
        ctx.save_for_backward(q, k, v, o, lse, plan)
        ctx.dims = dims
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        q, k, v, o, lse, plan = ctx.saved_tensors
        dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        dk = torch.empty(k.shape, dtype=q.dtype, device=q.device)
        dv = torch.empty(k.shape, dtype=q.dtype, device=q.device)
        if q.shape[0] == 0:
            return dq, dk, dv, None, None
        do = _rows(grad_output)
        with _lib.on_device(q.device):
            _lib.poll_status_eager(q.device)
            delta = torch.empty_like(lse)
            _lib.check(_lib.lib().mea_packed_attention_backward(
                ctypes.byref(ctx.dims), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), do.data_ptr(),
                do.stride(0), do.stride(1), lse.data_ptr(), plan.data_ptr(), plan.numel(), delta.data_ptr(),
                dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _lib.status_word(q.device),
                _lib.stream_ptr(q.device)))
            _lib.note_status_eager(q.device)
        return dq, dk, dv, None, None


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
    return PackedAttentionFunction.apply(q, k, v, cu_seqlens, float(q.shape[-1] ** -0.5 if scale is None else scale))
