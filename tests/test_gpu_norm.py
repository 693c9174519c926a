"""GPU: layer norm forward and backward, element by element against fp64.

Bounds.  u = finfo(type).eps / 2 is the final rounding.  Every fp32 sum adds at
most 128 terms one after the other on any path from a term to the total (a
thread's own elements, the lanes, the warps; for the weight's gradient a block's
rows, the groups, the partial rows), so it is off by at most F = 2^-17 of the sum
of magnitudes.  With X = |xhat| + (|x| + |mean|) rstd for what the statistics'
errors do to xhat:
  y:  u |y| + 4 F (|w| X + |b|)
  dx: u |dx| + 4 F rstd (|g| + mean|g| + X mean(|g| X))
  dw: u |dw| + 4 F sum |dy| X,   db: u |db| + 4 F sum |dy|
"""
import pytest
import torch

from gpu_util import DEV
from memory_efficient_attn_layer_b200 import LayerNorm, layer_norm

pytestmark = pytest.mark.gpu
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
F = 2.0 ** -17
TINY = {BF: 0.0, HF: 2.0 ** -25, FP: 0.0}


def _ref(x, w, b, eps, dy):
    x, dy = x.double(), dy.double()
    c = x.shape[-1]
    w64 = torch.ones(c, dtype=torch.float64, device=x.device) if w is None else w.double()
    b64 = torch.zeros(c, dtype=torch.float64, device=x.device) if b is None else b.double()
    mean = x.mean(-1, keepdim=True)
    rstd = ((x - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    xhat = (x - mean) * rstd
    g = dy * w64
    X = xhat.abs() + (x.abs() + mean.abs()) * rstd
    rows = tuple(range(x.dim() - 1))
    r = {"y": xhat * w64 + b64,
         "dx": rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True)),
         "dw": (dy * xhat).sum(rows), "db": dy.sum(rows)}
    bound = {"y": w64.abs() * X + b64.abs(),
             "dx": rstd * (g.abs() + g.abs().mean(-1, keepdim=True) + X * (g.abs() * X).mean(-1, keepdim=True)),
             "dw": (dy.abs() * X).sum(rows), "db": dy.abs().sum(rows)}
    return r, bound


def _run(x, w, b, eps, dy):
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w, b)]
    y = layer_norm(*leaves, eps)
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dy)
    out = {"y": y.detach()}
    out.update(zip([n for n, t in zip(("dx", "dw", "db"), leaves) if t is not None], grads))
    return out


def _check(x, w, b, eps, dy):
    got = _run(x, w, b, eps, dy)
    want, bound = _ref(x, w, b, eps, dy)
    for k, t in got.items():
        u = torch.finfo(t.dtype).eps / 2
        off = (t.double() - want[k]).abs()
        lim = u * want[k].abs() + 4 * F * (1 + u) * bound[k] + TINY[t.dtype]
        assert t.shape == want[k].shape and not bool((off > lim).any()), (k, float((off / lim.clamp_min(1e-300)).max()))
    return got


def _make(rows, c, dt, wdt, seed=0, weight=True, bias=True, offset=0.3):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = (torch.randn(rows, c, generator=g, device=DEV) + offset).to(dt)
    w = (1 + 0.2 * torch.randn(c, generator=g, device=DEV)).to(wdt) if weight else None
    b = (0.2 * torch.randn(c, generator=g, device=DEV)).to(wdt) if bias else None
    dy = torch.randn(rows, c, generator=g, device=DEV).to(dt)
    return x, w, b, dy


SIZES = [(1, 1), (3, 2), (5, 7), (1, 512), (64, 512), (33, 1001), (7, 100), (300, 2048), (17, 4096), (2500, 96),
         (1037, 1024), (9, 8192), (6, 5000), (5, 16384), (4, 10001), (3, 16392), (3, 20001)]


@pytest.mark.parametrize("rows,c", SIZES)
@pytest.mark.parametrize("dt,wdt", [(BF, BF), (BF, FP), (HF, HF), (HF, FP), (FP, FP)])
def test_sizes_and_types(rows, c, dt, wdt):
    _check(*_make(rows, c, dt, wdt, seed=c)[:3], 1e-5, _make(rows, c, dt, wdt, seed=c)[3])


@pytest.mark.parametrize("rows", [20000, 4097])
def test_many_rows(rows):
    x, w, b, dy = _make(rows, 768, BF, BF, seed=rows)
    _check(x, w, b, 1e-5, dy)


@pytest.mark.parametrize("rows,c,dt", [(9500, 512, BF), (4000, 1000, HF), (2500, 2048, BF), (1203, 2048, FP), (1001, 4096, BF),
                                       (700, 8192, HF), (601, 8192, FP), (600, 16384, BF), (450, 16384, FP),
                                       (20003, 17, BF), (9001, 100, HF), (9003, 333, FP), (6007, 1001, BF), (2501, 2047, HF),
                                       (1501, 4090, BF), (1201, 3001, FP), (1103, 6001, BF), (701, 8177, HF)])
def test_several_rounds_of_every_block(rows, c, dt):
    """More rows than the blocks take at a time, the last round a part of one: the rings of rows on their way go round."""
    _check(*_make(rows, c, dt, dt, seed=9)[:3], 1e-5, _make(rows, c, dt, dt, seed=10)[3])


@pytest.mark.parametrize("c,dt", [(16, BF), (17, BF), (23, HF), (31, BF), (9, FP), (11, FP), (4081, BF), (4082, HF), (8178, BF),
                                  (8185, BF), (4089, FP), (4093, FP)])
@pytest.mark.parametrize("rows", [1, 2, 7, 8, 9])
def test_widths_at_the_limits_of_the_vectors(rows, c, dt):
    """Rows at every alignment within 16 bytes, few of each."""
    x, w, b, dy = _make(rows, c, dt, dt, seed=rows * c)
    _check(x, w, b, 1e-5, dy)


@pytest.mark.parametrize("c", [64, 1001, 20001])
@pytest.mark.parametrize("weight,bias", [(True, False), (False, True), (False, False)])
def test_without_weight_or_bias(weight, bias, c):
    x, w, b, dy = _make(40, c, BF, BF, weight=weight, bias=bias)
    _check(x, w, b, 1e-5, dy)


def test_rows_far_off_centre():
    """mean / sd = 1000: the variance is summed about the mean."""
    x, w, b, dy = _make(50, 1024, FP, FP, seed=3, offset=1000.0)
    _check(x, w, b, 1e-5, dy)


def test_constant_rows():
    x = torch.full((6, 512), 3.0, device=DEV, dtype=BF)
    w, b = torch.full((512,), 2.0, device=DEV, dtype=BF), torch.linspace(-1, 1, 512, device=DEV).to(BF)
    assert torch.equal(layer_norm(x, w, b), b.expand(6, 512))
    assert bool(torch.isnan(layer_norm(x, w, b, eps=0.0)).all())  # 0 / 0, as the definition has it


@pytest.mark.parametrize("c", [256, 1001, 2048, 17000])
def test_a_row_with_nan_stays_alone(c):
    x, w, b, dy = _make(37, c, BF, BF, seed=5)
    clean = _run(x, w, b, 1e-5, dy)
    x[11, c // 2] = float("nan")
    got = _run(x, w, b, 1e-5, dy)
    rest = [i for i in range(37) if i != 11]
    for k in ("y", "dx"):
        assert torch.equal(got[k][rest], clean[k][rest]) and bool(torch.isnan(got[k][11]).all())
    assert torch.equal(got["db"], clean["db"]) and bool(torch.isnan(got["dw"]).all())


@pytest.mark.parametrize("layout", ["leading", "unaligned", "transposed", "broadcast_dy", "sliced"])
def test_shapes_and_strides(layout):
    x, w, b, dy = _make(60, 512, BF, BF, seed=6)
    want = _run(x, w, b, 1e-5, dy)
    if layout == "leading":
        x, dy = x.view(3, 4, 5, 512), dy.view(3, 4, 5, 512)
        want = {k: v.view(3, 4, 5, 512) if v.dim() == 2 else v for k, v in want.items()}
    elif layout == "unaligned":  # the scalar path: the same sums in another order, so to the bounds
        x, dy, w = (torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape) for t in (x, dy, w))
        _check(x, w, b, 1e-5, dy)
        return
    elif layout == "transposed":
        x, dy = x.t().contiguous().t(), dy.t().contiguous().t()
    elif layout == "broadcast_dy":
        dy = dy[:1].expand(60, 512)
        want = _run(x, w, b, 1e-5, dy.contiguous())
    else:
        x, dy = torch.cat([x, x], 1)[:, :512], torch.cat([dy, dy], 1)[:, :512]
    got = _run(x, w, b, 1e-5, dy)
    for k in got:
        assert torch.equal(got[k], want[k]), k


def test_no_rows():
    x, w, b, dy = _make(0, 256, BF, BF)
    got = _run(x, w, b, 1e-5, dy)
    assert got["y"].shape == (0, 256) and not bool(got["dw"].any()) and not bool(got["db"].any())


def test_same_call_same_bits():
    x, w, b, dy = _make(5000, 2048, BF, BF, seed=7)
    a, c = _run(x, w, b, 1e-5, dy), _run(x, w, b, 1e-5, dy)
    for k in a:
        assert torch.equal(a[k], c[k]), k


def test_needed_gradients_only():
    x, w, b, dy = _make(50, 512, BF, BF, seed=8)
    want = _run(x, w, b, 1e-5, dy)
    for which in range(3):
        leaves = [t.detach().requires_grad_(i == which) for i, t in enumerate((x, w, b))]
        (g,) = torch.autograd.grad(layer_norm(*leaves), leaves[which], dy)
        assert torch.equal(g, want[("dx", "dw", "db")[which]])


def test_captured_and_on_another_stream():
    x, w, b, dy = _make(100, 1024, BF, BF, seed=9)
    x2, dy2 = _make(100, 1024, BF, BF, seed=10)[0::3]
    want, want2 = _run(x, w, b, 1e-5, dy), _run(x2, w, b, 1e-5, dy2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _run(x, w, b, 1e-5, dy)
    torch.cuda.synchronize()
    assert all(torch.equal(got[k], want[k]) for k in got)
    xs, ds = x.clone(), dy.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _run(xs, w, b, 1e-5, ds)
    for a, d, ref in ((x2, dy2, want2), (x, dy, want)):
        xs.copy_(a)
        ds.copy_(d)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out[k], ref[k]) for k in out)


def test_directional_difference():
    """The gradient against a central difference of the forward itself, in fp32: loss = sum(y dy) along a direction.
    h = 2^-6: truncation h^2 / 6 times a third derivative of order the loss's own scale, rounding 2^-24 sum|y dy| / h."""
    x, w, b, dy = _make(16, 256, FP, FP, seed=11)
    got = _run(x, w, b, 1e-5, dy)
    g = torch.Generator(device=DEV).manual_seed(12)
    h = 2.0 ** -6
    for i, k in enumerate(("dx", "dw", "db")):
        d = torch.randn((x, w, b)[i].shape, generator=g, device=DEV)
        up, down = [x, w, b], [x, w, b]
        up[i], down[i] = up[i] + h * d, down[i] - h * d
        diff = float(((layer_norm(*up) - layer_norm(*down)).double() * dy.double()).sum()) / (2 * h)
        an = float((got[k].double() * d.double()).sum())
        scale = float((got["y"].double() * dy.double()).abs().sum())
        assert abs(diff - an) < (h * h + 2.0 ** -22 / h) * scale, k


def test_module():
    m = LayerNorm(384, device=DEV, dtype=BF)
    x = torch.randn(4, 9, 384, device=DEV).to(BF)
    assert torch.equal(m(x), layer_norm(x, m.weight, m.bias, 1e-5))
    assert [n for n, _ in LayerNorm(8, bias=False).named_parameters()] == ["weight"]


def test_arguments_are_checked():
    x, w, b, _ = _make(4, 64, BF, BF)
    for args, err in (((x, w[:3]), ValueError), ((x, w, b.float()), TypeError), ((x, w.half()), TypeError),
                      ((x.double(), None), TypeError), ((x, w, b, -1.0), ValueError), ((x, w, b, float("nan")), ValueError),
                      ((x[:, :0],), ValueError), ((x, w.cpu()), ValueError)):
        with pytest.raises(err):
            layer_norm(*args)
