"""The global norm of a list of gradients, and clipping by it: ``grad_norm`` and
``clip_grad_norm_`` (``mea_grad_norm``, ``mea_clip_grad_norm``).

For parameters that ``ShardedAdamW`` manages, whose gradients never appear in
``.grad``, give the optimizer ``max_grad_norm`` instead.
"""
from __future__ import annotations

from array import array
from typing import Iterable

import torch

from . import _lib

_KINDS = {2.0: 0, float("inf"): 1}


def _kind(norm_type) -> int:
    kind = _KINDS.get(float(norm_type))
    if kind is None:
        raise ValueError(f"norm_type must be 2 or inf, got {norm_type}")
    return kind


def _dense(tensors: list) -> tuple:
    """(the tensors, contiguous: the list itself where they all are already; their type codes)."""
    code = _lib.DTYPE_CODES.get
    codes = [code(t.dtype) for t in tensors]
    if None in codes or [t.layout for t in tensors].count(torch.strided) < len(tensors):
        t = next(t for t, c in zip(tensors, codes) if c is None or t.layout is not torch.strided)
        raise TypeError(f"gradients must be dense bf16, fp16 or fp32 tensors, got {t.dtype} ({t.layout})")
    if False in [t.is_contiguous() for t in tensors]:
        tensors = [t.contiguous() for t in tensors]
    return tensors, codes


def _arrays(tensors, codes):
    """(device index, arrays, (count, addresses of the arrays of pointers, element counts and type codes) for the C call)
    of contiguous tensors.  The arrays have to live until the call."""
    k, idx = len(tensors), tensors[0].get_device()
    if idx < 0:
        _lib.require_device(tensors[0].device)
    _lib.require_index(idx)
    if [t.get_device() for t in tensors].count(idx) < k:
        raise ValueError("all gradients must be on the same device")
    ptrs, ns = [t.data_ptr() for t in tensors], [t.numel() for t in tensors]
    if len(set(ptrs)) < k:  # tensors without elements have no address of their own
        held = [p for p, n in zip(ptrs, ns) if n]
        if len(set(held)) < len(held):
            raise ValueError("a gradient appears twice")
    arrays = array("Q", ptrs), array("q", ns), array("i", codes)
    return idx, arrays, (k, *[a.buffer_info()[0] for a in arrays])


def _workspace(like, k):
    """Workspace of a k-tensor call, on `like`'s device."""
    return torch.empty(_lib.lib().mea_grad_norm_workspace_size(k), dtype=torch.uint8, device=like.device)


def grad_norm(tensors: Iterable[torch.Tensor], norm_type: float = 2.0) -> torch.Tensor:
    """The norm of all elements of ``tensors`` as one vector: a 0-dim fp32 tensor on their device (no copy to the
    host).  ``norm_type`` 2 or inf.  An empty list has norm 0 (on the CPU)."""
    kind = _kind(norm_type)
    tensors, codes = _dense(list(tensors))
    if not tensors:
        return torch.tensor(0.0)
    idx, _held, args = _arrays(tensors, codes)
    out = torch.empty((), dtype=torch.float32, device=tensors[0].device)
    ws = _workspace(out, args[0])
    _lib.launch(idx, _lib.lib().mea_grad_norm, *args, kind, out.data_ptr(), None, ws.data_ptr(), ws.numel())
    return out


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Multiplies the gradients of ``parameters`` (a tensor or an iterable; those without ``.grad`` are passed over) in
    place by min(1, max_norm / (norm + 1e-6)), where norm is the global norm of them all, and returns that norm: a 0-dim
    fp32 tensor on their device.  torch.nn.utils.clip_grad_norm_'s rule, in two kernels over the whole list: one reads
    every gradient, the other scales, and does nothing where the norm is within max_norm.  The factor is applied in fp32
    and rounded to the gradient's type once.  ``error_if_nonfinite`` waits for the norm and raises before anything is
    scaled."""
    kind = _kind(norm_type)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must be >= 0, got {max_norm}")
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [g for g in (p.grad for p in parameters) if g is not None]
    if not grads:
        return torch.tensor(0.0)
    work, codes = _dense(grads)
    for g, w in zip(grads, work) if work is not grads else ():
        if g is not w and any(s == 0 and n > 1 for s, n in zip(g.stride(), g.shape)):
            raise ValueError("a gradient's elements share memory (an expanded tensor), so it cannot be scaled in place")
    idx, _held, args = _arrays(work, codes)
    if error_if_nonfinite:
        norm = grad_norm(work, norm_type)
        if not bool(torch.isfinite(norm)):
            raise RuntimeError(f"the total norm of order {norm_type} of the gradients is non-finite, so they cannot be clipped")
    out = torch.empty((), dtype=torch.float32, device=work[0].device)
    ws = _workspace(out, args[0])
    _lib.launch(idx, _lib.lib().mea_clip_grad_norm, *args, kind, max_norm, out.data_ptr(), ws.data_ptr(), ws.numel())
    for g, w in zip(grads, work) if work is not grads else ():
        if g is not w:
            with torch.no_grad():
                g.copy_(w)
    return out
