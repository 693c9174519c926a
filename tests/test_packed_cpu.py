"""CPU: the fp64 oracle of packed attention against finite differences and torch's autograd, and the refusals of
``packed_attention`` and of its C entry points before any device work."""
import ctypes
import math

import pytest
import torch

from memory_efficient_attn_layer_b200 import _lib, packed_attention
from oracle.packed import attention


def _inputs(lens, hq, hkv, n, seed=0):
    g = torch.Generator().manual_seed(seed)
    total = sum(lens)
    q, do = (torch.randn(total, hq, n, generator=g, dtype=torch.float64) for _ in range(2))
    k, v = (torch.randn(total, hkv, n, generator=g, dtype=torch.float64) for _ in range(2))
    cu = [0]
    for x in lens:
        cu.append(cu[-1] + x)
    return q, k, v, do, cu


@pytest.mark.parametrize("lens,hq,hkv,n", [([5, 0, 1, 9], 4, 2, 8), ([17], 3, 1, 16)])
def test_oracle_gradients_match_finite_differences(lens, hq, hkv, n):
    q, k, v, do, cu = _inputs(lens, hq, hkv, n)
    grads = attention(q, k, v, cu, do=do)
    g = torch.Generator().manual_seed(1)
    h = 1e-5

    def loss(*qkv):
        return float((attention(*qkv, cu)["o"] * do).sum())

    for i, name in enumerate(("dq", "dk", "dv")):
        d = torch.randn([q, k, v][i].shape, generator=g, dtype=torch.float64)
        up, down = [q, k, v], [q, k, v]
        up[i], down[i] = up[i] + h * d, down[i] - h * d
        want = (loss(*up) - loss(*down)) / (2 * h)
        # central difference: truncation h^2 times a third derivative of order 10^3 here, rounding 1e-13 / h
        assert abs(float((grads[name] * d).sum()) - want) < 1e-6 * max(1.0, abs(want)), name


def test_oracle_matches_autograd_of_the_definition():
    q, k, v, do, cu = _inputs([6, 11], 4, 2, 8, seed=3)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out = []
    for lo, hi in zip(cu, cu[1:]):
        kk, vv = (t[lo:hi].repeat_interleave(2, dim=1) for t in leaves[1:])
        s = torch.einsum("ihn,jhn->hij", leaves[0][lo:hi], kk) / math.sqrt(8)
        s = s.masked_fill(~torch.ones(hi - lo, hi - lo, dtype=torch.bool).tril(), -math.inf)
        out.append(torch.einsum("hij,jhn->ihn", s.softmax(-1), vv))
    o = torch.cat(out)
    want = torch.autograd.grad(o, leaves, do)
    got = attention(q, k, v, cu, do=do)
    assert torch.allclose(got["o"], o.detach(), rtol=0, atol=1e-12)
    for name, w in zip(("dq", "dk", "dv"), want):
        assert torch.allclose(got[name], w, rtol=0, atol=1e-12), name


def test_cpu_tensors_raise():
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        packed_attention(q, q, q, torch.tensor([0, 4], dtype=torch.int32))


def _dims(total=256, n_seqs=2, hq=8, hkv=2, n=64, dtype=0, scale=0.125, **strides):
    s = dict(q_row=hq * n, q_head=n, k_row=hkv * n, k_head=n, v_row=hkv * n, v_head=n)
    s.update(strides)
    return _lib.MeaPackedDims(total, n_seqs, hq, hkv, n, dtype, scale, *s.values())


@pytest.mark.parametrize("kw,code,text", [
    (dict(hq=8, hkv=3), 1, b"multiple of Hkv"),
    (dict(hq=0), 1, b"multiple of Hkv"),
    (dict(total=-1), 1, b"total=-1"),
    (dict(n_seqs=-2), 1, b"n_seqs=-2"),
    (dict(n=60), 2, b"multiple of 8"),
    (dict(n=136), 2, b"multiple of 8"),
    (dict(n=0), 2, b"multiple of 8"),
    (dict(dtype=2), 1, b"dtype 2"),
    (dict(scale=0.0), 1, b"scale"),
    (dict(scale=float("nan")), 1, b"scale"),
    (dict(scale=float("inf")), 1, b"scale"),
    (dict(total=2**30, hq=4096, hkv=4096), 2, b"too many tiles"), (dict(total=2**30 + 1), 2, b"2^30 rows"),
])
def test_sizes_are_refused(kw, code, text):
    L = _lib.lib()
    d = _dims(**kw)
    assert L.mea_packed_plan_size(ctypes.byref(d)) == 0
    assert text in L.mea_last_error_string()
    assert L.mea_packed_attention_forward(ctypes.byref(d), *[None] * 7, 0, None, None) == code
    assert L.mea_packed_attention_backward(ctypes.byref(d), *[None] * 5, 0, 0, None, None, 0, None, 0, *[None] * 5) == code
    assert L.mea_packed_backward_workspace_size(ctypes.byref(d)) == 0


def _fake(i):
    return 0x100000 * (i + 1)  # aligned stand-ins: the calls below never reach the device


@pytest.mark.parametrize("slot,value,code,text", [
    (0, None, 1, b"q is NULL"), (1, 0x7000008, 3, b"k must be 16-byte"), (2, 0x7000002, 3, b"v must be 16-byte"),
    (3, None, 1, b"cu_seqlens"), (4, 0x7000004, 3, b"o must be 16-byte"), (5, None, 1, b"lse2"), (6, None, 1, b"plan"),
    (5, 0x7000002, 3, b"4-byte"), (6, 0x7000010, 3, b"256-byte"),
])
def test_forward_refuses_bad_buffers_before_device_work(slot, value, code, text):
    L, d = _lib.lib(), _dims()
    args = [_fake(i) for i in range(7)]
    args[slot] = value
    need = L.mea_packed_plan_size(ctypes.byref(d))
    assert L.mea_packed_attention_forward(ctypes.byref(d), *args, need, None, None) == code
    assert text in L.mea_last_error_string()


@pytest.mark.parametrize("strides,text", [
    (dict(q_row=508), b"strides of q"), (dict(q_head=0), b"strides of q"), (dict(k_head=60), b"strides of k"),
    (dict(v_row=0), b"strides of v"), (dict(v_row=1 << 40), b"stride of v is too large"),
])
def test_forward_refuses_strides(strides, text):
    L, d = _lib.lib(), _dims(**strides)
    need = L.mea_packed_plan_size(ctypes.byref(d))
    assert L.mea_packed_attention_forward(ctypes.byref(d), *[_fake(i) for i in range(7)], need, None, None) in (2, 3)
    assert text in L.mea_last_error_string()


def test_small_plan_is_refused():
    L, d = _lib.lib(), _dims()
    need = L.mea_packed_plan_size(ctypes.byref(d))
    assert L.mea_packed_attention_forward(ctypes.byref(d), *[_fake(i) for i in range(7)], need - 1, None, None) == 7
    work = L.mea_packed_backward_workspace_size(ctypes.byref(d))
    for plan, ws in ((need - 1, work), (need, work - 1)):
        back = [_fake(i) for i in range(5)] + [512, 64, _fake(5), _fake(6), plan, _fake(7), ws] + [_fake(i) for i in range(8, 11)]
        assert L.mea_packed_attention_backward(ctypes.byref(d), *back, None, None) == 7


@pytest.mark.parametrize("slot,value,code,text", [
    (3, None, 1, b"o is NULL"), (4, 0x7000008, 3, b"dO must be 16-byte"), (5, 500, 3, b"strides of dO"),
    (7, None, 1, b"lse2"), (10, None, 1, b"workspace"), (10, 0x7000010, 3, b"256-byte"),
    (12, 0x7000008, 3, b"dq must be 16-byte"), (14, 0x7000008, 3, b"dv must be 16-byte"),
])
def test_backward_refuses_bad_buffers_before_device_work(slot, value, code, text):
    L, d = _lib.lib(), _dims()
    need = L.mea_packed_plan_size(ctypes.byref(d))
    work = L.mea_packed_backward_workspace_size(ctypes.byref(d))
    args = [_fake(i) for i in range(5)] + [512, 64, _fake(5), _fake(6), need, _fake(7), work] + [_fake(i) for i in range(8, 11)]
    args[slot] = value
    assert L.mea_packed_attention_backward(ctypes.byref(d), *args, None, None) == code
    assert text in L.mea_last_error_string()


def test_no_rows_is_nothing_to_do():
    L, d = _lib.lib(), _dims(total=0, n_seqs=3)
    assert L.mea_packed_attention_forward(ctypes.byref(d), *[None] * 7, 0, None, None) == 0
    assert L.mea_packed_attention_backward(ctypes.byref(d), *[None] * 5, 0, 0, None, None, 0, None, 0, *[None] * 5) == 0


def test_plan_holds_every_tile():
    """A header, and 16 bytes for each tile there can be of three lists: query tiles, key tiles, and the forward's items
    (one query tile each at these sizes)."""
    L = _lib.lib()
    for total, n_seqs, hq, hkv, tt in ((1000, 3, 8, 2, 32), (1000, 3, 2, 2, 128), (50, 200, 7, 1, 18), (64, 1, 256, 1, 1)):
        d = _dims(total=total, n_seqs=n_seqs, hq=hq, hkv=hkv)
        want = 16 * (2 * (total // tt + n_seqs) + total // 128 + n_seqs)
        assert want < L.mea_packed_plan_size(ctypes.byref(d)) <= want + 5 * 256
