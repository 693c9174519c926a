"""Layer norm with an affine weight and bias: ``layer_norm`` and ``LayerNorm``.

For the norms around the block (before an MLP, before the output projection);
the block's own input norm is part of ``fused_attn``.  The work is done by
``mea_layernorm_forward`` and ``mea_layernorm_backward``.
"""
from __future__ import annotations

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib


def _check(x, weight, bias, eps):
    _lib.require_device(x.device)
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"x must have a last dimension of at least one element, got shape {tuple(x.shape)}")
    if x.dtype not in _lib.DTYPE_CODES:
        raise TypeError(f"layer_norm computes on bf16, fp16 and fp32; got {x.dtype}")
    c = x.shape[-1]
    wtype = next((t.dtype for t in (weight, bias) if t is not None), x.dtype)
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if tuple(t.shape) != (c,):
            raise ValueError(f"{name} must be [{c}], got {tuple(t.shape)}")
        if t.dtype != wtype or t.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"weight and bias must both have x's type ({x.dtype}) or both be fp32; {name} is {t.dtype}")
        if t.device != x.device:
            raise ValueError("all tensors must be on the same device")
    if not 0.0 <= eps < 3e38:
        raise ValueError(f"eps must be >= 0 and finite, got {eps}")
    return wtype


def _forward(x, weight, bias, eps):
    """(y, (x, weight, row statistics), type codes, weight type)."""
    dt, idx, c = x.dtype, x.get_device(), x.shape[-1] if x.dim() else 0
    wtype = dt if weight is None else weight.dtype
    if not (idx >= 0 and dt in _lib.DTYPE_CODES and c > 0 and 0.0 <= eps < 3e38 and (wtype is dt or wtype is torch.float32)
            and weight is not None and weight.get_device() == idx and weight.dim() == 1 and weight.shape[0] == c
            and (bias is None or (bias.dtype is wtype and bias.get_device() == idx and bias.dim() == 1
                                  and bias.shape[0] == c))):
        wtype = _check(x, weight, bias, eps)
    _lib.require_index(idx)
    x = x.contiguous()
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    rows = x.numel() // c
    y = torch.empty_like(x)
    stats = torch.empty(2 * rows, dtype=torch.float32, device=x.device)
    codes = _lib.DTYPE_CODES[dt], _lib.DTYPE_CODES[wtype]
    at = stats.data_ptr()
    _lib.launch(idx, _lib.lib().mea_layernorm_forward, rows, c, eps, *codes, x.data_ptr(), _lib.ptr(weight), _lib.ptr(bias),
                y.data_ptr(), at, at + 4 * rows)
    return y, (x, weight, stats), codes, wtype


def _backward(ctx, dy):
    x, weight, stats = ctx.saved_tensors
    dy = dy.contiguous()
    c = x.shape[-1]
    rows = x.numel() // c
    dx = torch.empty_like(x)
    dw, db = (x.new_empty(c, dtype=ctx.wtype) if need else None for need in ctx.needs_input_grad[1:3])
    L = _lib.lib()
    ws, nbytes = None, 0
    if dw is not None or db is not None:
        nbytes = L.mea_layernorm_workspace_size(rows, c)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    at = stats.data_ptr()
    _lib.launch(x.get_device(), L.mea_layernorm_backward, rows, c, *ctx.codes, dy.data_ptr(), x.data_ptr(), _lib.ptr(weight),
                at, at + 4 * rows, dx.data_ptr(), _lib.ptr(dw), _lib.ptr(db), _lib.ptr(ws), nbytes)
    return dx, dw, db, None


_backward_once = once_differentiable(_backward)


class LayerNormFunction(torch.autograd.Function):
    """Autograd node of ``layer_norm``.  Kept for the backward: x, the weight and each row's mean and 1/sd (fp32)."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, saved, ctx.codes, ctx.wtype = _forward(x, weight, bias, eps)
        ctx.save_for_backward(*saved)
        return y

    @staticmethod
    def backward(ctx, dy):
        # The gradients have no derivative of their own; the marking costs host time, so only where one could be taken.
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, dy)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over x's last dimension.

    x: bf16, fp16 or fp32, any shape and width; weight and bias: [C], of x's type or fp32, either may be None.  The sums
    (row statistics, and the gradients of weight and bias over the rows) are fp32, in a fixed order."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return LayerNormFunction.apply(x, weight, bias, float(eps))
    return _forward(x, weight, bias, float(eps))[0]


class LayerNorm(nn.Module):
    """``layer_norm`` with its parameters: weight one, bias zero (none with ``bias=False``)."""

    def __init__(self, dim: int, eps: float = 1e-5, bias: bool = True, device=None, dtype=None):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim, device=device, dtype=dtype))
        self.bias = nn.Parameter(torch.zeros(dim, device=device, dtype=dtype)) if bias else None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return layer_norm(x, self.weight, self.bias, self.eps)
