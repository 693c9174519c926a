"""GPU: the global gradient norm, clipping by it, and ShardedAdamW's max_grad_norm.

Bounds.  The norm: squares are summed in fp32 over at most 8 values and in fp64
after that, so its square is off by at most 8 * 2^-24 relative and the norm by half
of that, plus the final rounding: 2^-21.  A scaled element: one fp32 product with
a factor that is off by 2^-21 and rounded to fp32, then the rounding u = eps / 2 of
its type (and half of fp16's smallest subnormal): u + 2^-20.
"""
import math

import numpy as np
import pytest
import torch

from gpu_util import DEV
from memory_efficient_attn_layer_b200 import MeaError, ShardedAdamW, clip_grad_norm_, grad_norm
from oracle.adamw import adamw_step

pytestmark = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _params(shapes, dts, seed=0, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    ps = []
    for i, s in enumerate(shapes):
        p = torch.nn.Parameter(torch.zeros(s, device=DEV, dtype=dts[i % len(dts)]))
        p.grad = (torch.randn(s, generator=g, device=DEV) * scale).to(p.dtype)
        ps.append(p)
    return ps


def _norm64(ts):
    return math.sqrt(sum(float(t.double().square().sum()) for t in ts))


def _check(ps, max_norm):
    before = [p.grad.clone() for p in ps]
    want = _norm64(before)
    got = clip_grad_norm_(ps, max_norm)
    assert got.dtype == torch.float32 and got.dim() == 0
    assert abs(float(got) - want) <= 2.0 ** -21 * want
    f = min(1.0, max_norm / (want + 1e-6))
    for p, b in zip(ps, before):
        ref = b.double() * f
        u = torch.finfo(p.dtype).eps / 2
        assert bool(((p.grad.double() - ref).abs() <= (u + 2.0 ** -20) * ref.abs() + (2.0 ** -25 if p.dtype == HF else 0.0)).all())
    return before


@pytest.mark.parametrize("dts", [[BF], [HF], [FP], [BF, FP, HF]])
@pytest.mark.parametrize("shapes", [[(1,)], [(7,), (3, 5), (1001,)], [(512, 512)] * 5, [(32768,), (32769,), (65535,), (2,)],
                                    [(1500, 1001), (9,)]])
@pytest.mark.parametrize("max_norm", [0.25, 0.0])
def test_norm_and_clip(shapes, dts, max_norm):
    _check(_params(shapes, dts, seed=len(shapes)), max_norm)


def test_more_tensors_than_one_launch_takes():
    shapes = [(1 + 37 * i % 999,) for i in range(1300)]
    _check(_params(shapes, [BF, FP, HF], seed=4), 1.0)


def test_within_the_threshold_every_bit_stays():
    ps = _params([(300, 7), (1000,)], [BF, FP, HF], scale=0.001)
    before = [p.grad.clone() for p in ps]
    clip_grad_norm_(ps, 1.0)
    assert all(torch.equal(p.grad, b) for p, b in zip(ps, before))


@pytest.mark.parametrize("dt", [BF, HF, FP])
def test_views_at_odd_offsets(dt):
    """Gradients that start and end between 16-byte boundaries; their neighbours in the buffer stay."""
    flat = torch.randn(5000, device=DEV).to(dt)
    keep = flat.clone()
    ps, inside = [], torch.zeros(5000, dtype=torch.bool, device=DEV)
    for lo, n in ((1, 3), (5, 1), (9, 64), (101, 1000), (1103, 999), (2222, 0), (2300, 2500)):
        p = torch.nn.Parameter(torch.zeros(n, device=DEV, dtype=dt))
        p.grad = flat[lo:lo + n]
        inside[lo:lo + n] = True
        ps.append(p)
    _check(ps, 0.5)
    assert torch.equal(flat[~inside], keep[~inside]) and not torch.equal(flat[inside], keep[inside])


def test_strided_gradients():
    p, q = (torch.nn.Parameter(torch.zeros(40, 30, device=DEV)) for _ in range(2))
    p.grad = torch.randn(30, 40, device=DEV).t()
    q.grad = torch.randn(40, 60, device=DEV)[:, ::2]
    _check([p, q], 0.5)


@pytest.mark.parametrize("scale", [1e25, 1e-25, 1e-38])
def test_squares_outside_fp32(scale):
    ps = _params([(1000,), (37,)], [FP, BF], scale=scale)
    want = _norm64([p.grad for p in ps])
    assert abs(float(grad_norm([p.grad for p in ps])) - want) <= 2.0 ** -21 * want + 1e-45
    if scale > 1:
        _check(ps, 2.0)


def test_inf_norm_and_nonfinite():
    ps = _params([(100, 33), (7,)], [FP, BF], seed=2)
    want = max(float(p.grad.abs().max()) for p in ps)
    assert float(grad_norm([p.grad for p in ps], float("inf"))) == want
    before = [p.grad.clone() for p in ps]
    assert float(clip_grad_norm_(ps, 0.5, float("inf"))) == want
    for p, b in zip(ps, before):
        ref = b.double() * (0.5 / (want + 1e-6))
        assert bool(((p.grad.double() - ref).abs() <= (torch.finfo(p.dtype).eps / 2 + 2.0 ** -20) * ref.abs()).all())
    for value in (float("nan"), float("inf")):
        ps = _params([(100,), (7,)], [FP, BF], seed=3)
        ps[1].grad[3] = value
        before = [p.grad.clone() for p in ps]
        with pytest.raises(RuntimeError, match="non-finite"):
            clip_grad_norm_(ps, 1.0, error_if_nonfinite=True)
        assert all(torch.equal(p.grad.nan_to_num(7.0), b.nan_to_num(7.0)) for p, b in zip(ps, before))
        for kind in (2.0, float("inf")):
            got = float(grad_norm([p.grad for p in ps], kind))
            assert got == value or (math.isnan(got) and math.isnan(value))
        clip_grad_norm_(ps, 1.0)  # as torch's rule has it: times NaN, or times zero
        assert bool(torch.isnan(ps[1].grad[3])) and (bool(torch.isnan(ps[0].grad).all()) or not bool(ps[0].grad.any()))


def test_matches_torch():
    shapes = [(64, 64), (100,), (3, 5, 7)]
    a, b = _params(shapes, [FP], seed=5), _params(shapes, [FP], seed=5)
    na, nb = clip_grad_norm_(a, 1.5), torch.nn.utils.clip_grad_norm_(b, 1.5)
    assert abs(float(na) - float(nb)) <= 1e-6 * float(nb)
    for p, q in zip(a, b):
        assert torch.allclose(p.grad, q.grad, rtol=2e-6, atol=0)


def test_nothing_to_clip():
    p = torch.nn.Parameter(torch.zeros(3, device=DEV))
    assert float(clip_grad_norm_([p], 1.0)) == 0.0 and float(clip_grad_norm_([], 1.0)) == 0.0
    p.grad = torch.zeros(3, device=DEV)
    q = torch.nn.Parameter(torch.zeros(0, device=DEV))
    q.grad = torch.zeros(0, device=DEV)
    assert float(clip_grad_norm_([p, q], 1.0)) == 0.0 and float(clip_grad_norm_(q, 1.0)) == 0.0
    assert not bool(p.grad.any())


def test_refusals():
    p = _params([(10,)], [FP])[0]
    q = torch.nn.Parameter(torch.zeros(10, device=DEV))
    q.grad = p.grad
    with pytest.raises(ValueError, match="twice"):
        clip_grad_norm_([p, q], 1.0)
    with pytest.raises(ValueError, match="norm_type"):
        clip_grad_norm_([p], 1.0, 3.0)
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            clip_grad_norm_([p], bad)
    with pytest.raises(TypeError):
        grad_norm([p.grad.double()])
    with pytest.raises(TypeError):
        grad_norm([torch.zeros(3, device=DEV).to_sparse()])
    with pytest.raises(RuntimeError, match="CUDA"):
        grad_norm([torch.zeros(3)])
    with pytest.raises(ValueError, match="device"):
        grad_norm([p.grad, torch.zeros(3)])


def test_same_bits_capture_and_streams():
    shapes = [(512, 512)] * 5 + [(999,)] * 20
    a = _params(shapes, [BF, FP], seed=6)
    want_norm = clip_grad_norm_(a, 1.0)
    want = [p.grad.clone() for p in a]
    s = torch.cuda.Stream()
    b = _params(shapes, [BF, FP], seed=6)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        got = clip_grad_norm_(b, 1.0)
    torch.cuda.synchronize()
    assert torch.equal(got, want_norm) and all(torch.equal(p.grad, w) for p, w in zip(b, want))
    c = _params(shapes, [BF, FP], seed=6)
    raw = [p.grad.clone() for p in c]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_grad_norm_(c, 1.0)
    for _ in range(3):
        for p, r in zip(c, raw):
            p.grad.copy_(r)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, want_norm) and all(torch.equal(p.grad, w) for p, w in zip(c, want))


@pytest.mark.parametrize("max_norm", [0.5, 1e6])
def test_sharded_adamw_clips(max_norm):
    hp = dict(lr=1e-2, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=1e-2)
    g = torch.Generator(device=DEV).manual_seed(1)
    ws = [torch.nn.Parameter(torch.randn(s, generator=g, device=DEV).to(BF)) for s in ((65, 33), (1000,), (8, 8))]
    opt = ShardedAdamW(ws, lr=hp["lr"], weight_decay=hp["weight_decay"], max_grad_norm=max_norm)
    master = [w.detach().float().cpu().numpy().ravel().copy() for w in ws]
    m, v = ([np.zeros_like(x) for x in master] for _ in range(2))
    for step in (1, 2):
        opt.zero_grad()
        for w in ws:
            w.grad = (torch.randn(w.shape, generator=g, device=DEV) * 3).to(BF)
        grads = [w.grad.float() for w in ws]
        norm = _norm64(grads)
        opt.step()
        assert abs(float(opt.grad_norm) - norm) <= 2.0 ** -21 * norm
        f = min(1.0, max_norm / (norm + 1e-6))
        for i, gr in enumerate(grads):
            adamw_step(master[i], m[i], v[i], gr.cpu().numpy().ravel(), step=step, grad_scale=f, **hp)
        got = [opt.master[o:o + w.numel()].cpu().numpy() for w, o in zip(ws, opt.layout.offsets)]
        for a, b in zip(got, master):
            np.testing.assert_allclose(a, b, rtol=1e-5, atol=2e-6)
    plain = ShardedAdamW([torch.nn.Parameter(torch.zeros(8, device=DEV, dtype=BF))])
    plain.step()
    assert plain.grad_norm is None
    with pytest.raises(ValueError, match="max_grad_norm"):
        ShardedAdamW([torch.nn.Parameter(torch.zeros(8, device=DEV, dtype=BF))], max_grad_norm=-1.0)


def test_gradients_that_share_memory_are_refused():
    buf = torch.randn(300, device=DEV)
    keep = buf.clone()
    p, q = (torch.nn.Parameter(torch.zeros(200, device=DEV)) for _ in range(2))
    p.grad, q.grad = buf[:200], buf[100:]
    with pytest.raises(MeaError, match="overlap"):
        clip_grad_norm_([p, q], 1e-3)
    q.grad = buf[:1].expand(200)
    with pytest.raises(ValueError, match="share memory"):
        clip_grad_norm_([p, q], 1e-3)
    assert torch.equal(buf, keep)
