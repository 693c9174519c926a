"""GPU: one training step on packed documents, as a caller puts the pieces together: layer norm, projections, rotary by
position within the document, packed attention with grouped heads, a residual MLP, a loss over the real rows, backward,
clipping by the global norm, AdamW.  Checked against the same model in fp32 plain PyTorch on the same (bf16) parameters
at the bars of the residual-stack test: outputs max|a-b| / max|b| <= 3e-2 over two layers, gradient cosine > 0.999."""
import math

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from gpu_util import DEV, cos, maxrel
from memory_efficient_attn_layer_b200 import (LayerNorm, ShardedAdamW, Yarn, check_device_status, clip_grad_norm_, layer_norm,
                                              packed_attention)
from oracle.adamw import adamw_step

pytestmark = pytest.mark.gpu
C, HQ, HKV, N, LAYERS = 256, 4, 2, 64, 2


def _swap(x):
    return x.reshape(*x.shape[:-1], -1, 2).flip(-1).reshape(x.shape)


class Layer(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.norm1, self.norm2 = LayerNorm(C), LayerNorm(C, bias=False)
        self.qkv = torch.nn.Linear(C, (HQ + 2 * HKV) * N, bias=False)
        self.o = torch.nn.Linear(HQ * N, C, bias=False)
        self.up, self.down = torch.nn.Linear(C, 4 * C, bias=False), torch.nn.Linear(4 * C, C, bias=False)

    def forward(self, x, cu, f1, f2, ops):
        norm, attend = ops
        h = norm(x, self.norm1.weight, self.norm1.bias)
        q, k, v = self.qkv(h).view(-1, HQ + 2 * HKV, N).split([HQ, HKV, HKV], dim=1)
        q, k = (t * f1 + _swap(t) * f2 for t in (q, k))
        x = x + self.o(attend(q, k, v, cu).reshape(-1, HQ * N))
        h = norm(x, self.norm2.weight, None)
        return x + self.down(F.relu(self.up(h)).square())


def _plain_norm(x, w, b):
    return F.layer_norm(x, (C,), w, b)


def _plain_attend(q, k, v, cu):
    out = []
    for lo, hi in zip(cu.tolist(), cu.tolist()[1:]):
        kk, vv = (t[lo:hi].repeat_interleave(HQ // HKV, dim=1) for t in (k, v))
        s = torch.einsum("ihn,jhn->hij", q[lo:hi], kk) / math.sqrt(N)
        s = s.masked_fill(~torch.ones(hi - lo, hi - lo, dtype=torch.bool, device=q.device).tril(), -math.inf)
        out.append(torch.einsum("hij,jhn->ihn", s.softmax(-1), vv))
    out.append(torch.zeros(q.shape[0] - cu.tolist()[-1], HQ, N, device=q.device))
    return torch.cat(out)


def _setup(seed=0, pad=9):
    torch.manual_seed(seed)
    lens = [130, 1, 301, 64, 128]
    cu = torch.tensor([0] + np.cumsum(lens).tolist(), dtype=torch.int32, device=DEV)
    real = sum(lens)
    layers = torch.nn.ModuleList(Layer() for _ in range(LAYERS)).to(device=DEV, dtype=torch.bfloat16)
    for m in layers.modules():
        if isinstance(m, LayerNorm):
            m.weight.data += 0.1 * torch.randn_like(m.weight)
    pos = torch.cat([torch.arange(n) for n in lens] + [torch.zeros(pad, dtype=torch.long)]).to(DEV)
    yarn = Yarn(N, 512, device=DEV)
    f1, f2 = yarn.factor1[pos][:, None], yarn.factor2[pos][:, None]
    x = torch.randn(real + pad, C, device=DEV).to(torch.bfloat16)
    dy = torch.randn(real, C, device=DEV).to(torch.bfloat16)
    return layers, cu, f1, f2, x, dy, real


def _forward(layers, x, cu, f1, f2, ops):
    for layer in layers:
        x = layer(x, cu, f1, f2, ops)
    return x


def test_step_matches_fp32():
    layers, cu, f1, f2, x, dy, real = _setup()
    xb = x.clone().requires_grad_(True)
    y = _forward(layers, xb, cu, f1, f2, (layer_norm, packed_attention))
    y[:real].backward(dy)
    import copy

    ref = copy.deepcopy(layers).float()
    for p in ref.parameters():
        p.grad = None
    xr = x.float().requires_grad_(True)
    yr = _forward(ref, xr, cu, f1.float(), f2.float(), (_plain_norm, _plain_attend))
    yr[:real].backward(dy.float())
    assert maxrel(y[:real].detach().float(), yr[:real].detach()) <= 3e-2
    assert cos(xb.grad[:real].float(), xr.grad[:real]) > 0.999
    assert not bool(xb.grad[real:].any())  # rows that no document owns
    for (name, p), q in zip(layers.named_parameters(), ref.parameters()):
        assert cos(p.grad.float(), q.grad) > 0.999, name
    # clipping these gradients: the norm, and every gradient times the factor
    grads = [p.grad.clone() for p in layers.parameters()]
    want = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    norm = clip_grad_norm_(layers.parameters(), 0.1 * want)
    assert abs(float(norm) - want) <= 2.0 ** -21 * want
    f = 0.1 * want / (want + 1e-6)
    for p, g in zip(layers.parameters(), grads):
        ref_g = g.double() * f
        assert bool(((p.grad.double() - ref_g).abs() <= (2.0 ** -8 + 2.0 ** -20) * ref_g.abs()).all())
    check_device_status(DEV)


def test_documents_do_not_see_each_other():
    """The other documents' rows change, this one's outputs and input gradients keep their bits."""
    layers, cu, f1, f2, x, dy, real = _setup(seed=1)
    lo, hi = int(cu[2]), int(cu[3])
    got = []
    for other in (1.0, -3.0):
        x2 = x * other
        x2[lo:hi] = x[lo:hi]
        x2 = x2.detach().requires_grad_(True)
        y = _forward(layers, x2, cu, f1, f2, (layer_norm, packed_attention))
        (g,) = torch.autograd.grad(y[:real], x2, dy)
        got.append((y[lo:hi].detach(), g[lo:hi]))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


def test_sharded_adamw_step_with_clipping():
    layers, cu, f1, f2, x, dy, real = _setup(seed=2)
    params = list(layers.parameters())
    before = [p.detach().float().cpu().numpy().ravel().copy() for p in params]
    opt = ShardedAdamW(params, lr=1e-2, weight_decay=0.0, max_grad_norm=1.0)
    y = _forward(layers, x, cu, f1, f2, (layer_norm, packed_attention))
    y[:real].backward(dy)
    grads = [p.grad.float() for p in params]
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    opt.step()
    assert abs(float(opt.grad_norm) - norm) <= 2.0 ** -21 * norm and norm > 1.0
    for p, b, g, o in zip(params, before, grads, opt.layout.offsets):
        m, v = np.zeros_like(b), np.zeros_like(b)
        adamw_step(b, m, v, g.cpu().numpy().ravel(), lr=1e-2, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, step=1,
                   grad_scale=1.0 / (norm + 1e-6))
        np.testing.assert_allclose(opt.master[o:o + p.numel()].cpu().numpy(), b, rtol=1e-5, atol=2e-6)


def test_captured_step():
    """Forward, backward and clipping in one graph, replayed on other rows and other documents."""
    layers, cu, f1, f2, x, dy, real = _setup(seed=3)
    params = list(layers.parameters())
    x2 = torch.randn(x.shape, device=DEV).to(x.dtype)
    cu2 = torch.tensor([0, 5, 5, 400, 500, real], dtype=torch.int32, device=DEV)

    def step(rows, lens):
        y = _forward(layers, rows, lens, f1, f2, (layer_norm, packed_attention))
        for p, g in zip(params, torch.autograd.grad(y[:real], params, dy)):
            p.grad = g
        return y.detach(), clip_grad_norm_(params, 1.0)

    want = []
    for rows, lens in ((x, cu), (x2, cu2)):
        y, norm = step(rows, lens)
        want.append((y, norm, [p.grad.clone() for p in params]))
    rows, lens = x.clone(), cu.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, norm = step(rows, lens)
        grads = [p.grad for p in params]
    for i, (a, b) in ((1, (x2, cu2)), (0, (x, cu)), (1, (x2, cu2))):
        rows.copy_(a)
        lens.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[i][0]) and torch.equal(norm, want[i][1])
        assert all(torch.equal(g, w) for g, w in zip(grads, want[i][2]))
