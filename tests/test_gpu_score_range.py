"""GPU: the block's attention kernels on scores that lie more than 127 log2 units apart within a row: their weights
are zero, and the outputs and gradients stay finite and right."""
import math

import pytest
import torch

from gpu_util import DEV, P, bf16, call, cos, maxrel, status, stream

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N", [32, 64, 128])
def test_attention_with_scores_far_apart(N):
    B, H, T = 1, 2, 256
    g = torch.Generator().manual_seed(N)
    # scores of standard deviation 100 (natural units)
    q, k = (bf16(torch.randn(B, H, T, N, generator=g) * 10) for _ in range(2))
    v, do = (bf16(torch.randn(B, H, T, N, generator=g)) for _ in range(2))
    gs = torch.ones_like(v)
    gated = torch.empty(B, T, H * N, dtype=torch.bfloat16, device=DEV)
    o = torch.empty_like(v)
    lse = torch.empty(B, H, T, device=DEV)
    s = status()
    call("mea_attention_forward", B, H, T, N, P(q), P(k), P(v), P(gs), P(gated), P(lse), P(o), P(s), stream(), status_buf=s)
    qf, kf, vf = (t.double().requires_grad_(True) for t in (q, k, v))
    sc = (qf @ kf.transpose(-1, -2)) / math.sqrt(N)
    want = sc.masked_fill(~torch.ones(T, T, dtype=torch.bool, device=DEV).tril(), -math.inf).softmax(-1) @ vf
    assert bool(torch.isfinite(o).all())
    assert maxrel(o, want.detach()) < 2e-2
    want.backward(do.double())
    delta = (do.float() * o.float()).sum(-1).contiguous()
    dq = torch.zeros(B, H, T, N, device=DEV)
    dk = torch.empty_like(k)
    dv = torch.empty(B, T, H * N, dtype=torch.bfloat16, device=DEV)
    call("mea_attention_backward", B, H, T, N, P(q), P(k), P(v), P(do), P(lse), P(delta), P(dq), P(dk), P(dv), H * N,
         P(s), stream(), status_buf=s)
    for got, ref in ((dq, qf.grad), (dk, kf.grad), (dv.view(B, T, H, N).transpose(1, 2), vf.grad)):
        assert bool(torch.isfinite(got).all())
        assert cos(got, ref) > 0.999
