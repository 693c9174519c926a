"""GPU: packed causal attention with grouped heads, forward and backward, element by element against the fp64 oracle
within the bounds that oracle/packed.py derives from the roundings, and the calls around it (padding, strides, streams,
captures, refusals)."""
import pytest
import torch

from gpu_util import DEV
from memory_efficient_attn_layer_b200 import MeaError, check_device_status, packed_attention
from oracle.packed import attention

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
TINY = {BF: 0.0, HF: 2.0 ** -25}


def _make(lens, hq, hkv, n, dt, seed=0, before=0, behind=0, joint=True):
    g = torch.Generator(device=DEV).manual_seed(seed)
    cu = [before]
    for x in lens:
        cu.append(cu[-1] + x)
    total = cu[-1] + behind
    if joint:
        t = torch.randn(total, hq + 2 * hkv, n, generator=g, device=DEV).to(dt)
        q, k, v = t.split([hq, hkv, hkv], dim=1)
    else:
        q, k, v = (torch.randn(total, h, n, generator=g, device=DEV).to(dt) for h in (hq, hkv, hkv))
    do = torch.randn(total, hq, n, generator=g, device=DEV).to(dt)
    return q, k, v, do, cu


def _run(q, k, v, do, cu, scale=None):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    o = packed_attention(*leaves, torch.tensor(cu, dtype=torch.int32, device=DEV), scale)
    grads = torch.autograd.grad(o, leaves, do)
    torch.cuda.synchronize()
    check_device_status(DEV)
    return dict(zip(("o", "dq", "dk", "dv"), (o.detach(), *grads)))


def _compare(got, want, skip=()):
    for x in ("o", "dq", "dk", "dv"):
        if x in skip:
            continue
        off = (got[x].double() - want[x]).abs()
        over = off > want["b" + x]
        assert not bool(over.any()), (f"{x}: {int(over.sum())} of {over.numel()} elements out of bounds, worst "
                                      f"{float((off / want['b' + x].clamp_min(1e-300)).max()):.3g} times")
        # and far inside them on the whole: roundings are independent, so their 2-norm is a fraction of the bound's
        assert float(off.norm()) <= 0.5 * float(want["b" + x].norm()) + 1e-30, x


def _check(lens, hq, hkv, n, dt, scale=None, **kw):
    q, k, v, do, cu = _make(lens, hq, hkv, n, dt, **kw)
    got = _run(q, k, v, do, cu, scale)
    _compare(got, attention(q, k, v, cu, scale, do, torch.finfo(dt).eps, TINY[dt]))
    return got, cu


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("n", [64, 128])
@pytest.mark.parametrize("lens", [[1], [0, 1, 0], [2], [127], [128], [129], [256], [1, 127, 128, 129, 0, 300, 5]])
def test_lengths(lens, n, dt):
    _check(lens, 4, 2, n, dt, seed=len(lens) + n)


@pytest.mark.parametrize("n", [8, 32, 40, 56, 72, 80, 96, 120])
def test_head_dims(n):
    _check([200, 3, 131], 3, 3, n, BF, seed=n)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (6, 2), (7, 1), (8, 1), (12, 2), (16, 2), (48, 1), (71, 1), (256, 1), (30, 10)])
@pytest.mark.parametrize("n", [64, 128])
def test_head_groups(hq, hkv, n):
    _check([150, 1, 33, 260], hq, hkv, n, BF, seed=hq)


@pytest.mark.parametrize("n,hq,hkv", [(64, 8, 8), (128, 4, 1)])
def test_long_and_ragged(n, hq, hkv):
    _check([2048, 1100, 3, 777, 1, 4500, 640], hq, hkv, n, BF, seed=5)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("lens,hq,hkv,n", [([3000], 8, 1, 128), ([1500, 1, 700, 129], 7, 1, 64), ([2000, 40, 333], 4, 2, 80),
                                           ([900], 256, 1, 64)])
def test_walks_cut_into_parts(lens, hq, hkv, n, dt):
    """Few key tiles and long walks: dK and dV come in parts that are added at the end."""
    _check(lens, hq, hkv, n, dt, seed=21, before=3, behind=50)


def test_many_sequences():
    """More sequences and tiles than the plan's block has threads."""
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 4, (2500,), generator=g).tolist()
    _check(lens, 2, 1, 64, BF, seed=9)


@pytest.mark.parametrize("n,hq,hkv", [(128, 8, 8), (128, 16, 8), (64, 16, 16)])
def test_tiles_taken_by_sequence(n, hq, hkv):
    """K and V beyond half of L2 and many tiles: sequence after sequence instead of the longest tiles first."""
    _check([300, 257, 0, 256, 310] * 30 + [1000, 1, 2000, 700], hq, hkv, n, BF, seed=17, behind=7)


@pytest.mark.parametrize("dt", [BF, HF])
def test_scale_and_large_scores(dt):
    _check([190, 40], 2, 2, 64, dt, scale=0.5, seed=2)


def test_scores_that_grow_along_the_row():
    """Later keys score higher: the running maximum moves in every key tile."""
    q, k, v, do, cu = _make([700], 2, 1, 64, BF, seed=4, joint=False)
    k = (k.float() * torch.linspace(0.1, 2.0, 700, device=DEV)[:, None, None]).to(BF)
    got = _run(q, k, v, do, cu, 0.3)
    _compare(got, attention(q, k, v, cu, 0.3, do, torch.finfo(BF).eps))


@pytest.mark.parametrize("n", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(2, 2), (7, 1), (8, 2)])
def test_rows_outside_the_sequences(n, hq, hkv):
    """Rows before the first and behind the last sequence hold NaN everywhere; they give zeros and disturb nothing."""
    lens = [70, 0, 130, 61]
    q, k, v, do, cu = _make(lens, hq, hkv, n, BF, seed=8, before=37, behind=150)
    want = attention(q, k, v, cu, None, do, torch.finfo(BF).eps)
    for t in (q, k, v, do):
        t[:cu[0]] = float("nan")
        t[cu[-1]:] = float("nan")
    got = _run(q, k, v, do, cu)
    for x in got.values():
        assert not bool(x[:cu[0]].any()) and not bool(x[cu[-1]:].any())
    _compare(got, want)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("n", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(2, 2), (7, 1), (16, 2)])
def test_another_sequence_with_nonfinite_values(n, hq, hkv, value):
    """Sequence 1 of 3 holds inf or NaN in q, k, v and do: the others' outputs and gradients keep their bits."""
    q, k, v, do, cu = _make([77, 150, 201], hq, hkv, n, BF, seed=11)
    clean = _run(q, k, v, do, cu)
    for t in (q, k, v, do):
        t[cu[1]:cu[2]] = value
    got = _run(q, k, v, do, cu)
    for x in got:
        for lo, hi in ((cu[0], cu[1]), (cu[2], cu[3])):
            assert torch.equal(got[x][lo:hi], clean[x][lo:hi]), x


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("n", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(2, 2), (7, 1), (8, 1)])
def test_causal_whatever_later_rows_hold(n, hq, hkv, value):
    """k and v from row 90 on hold inf or NaN: o before it keeps its bits; with v alone o from there on is non-finite in
    the columns that hold the value."""
    q, k, v, do, cu = _make([200, 64], hq, hkv, n, BF, seed=12)
    cut = torch.tensor(cu, dtype=torch.int32, device=DEV)
    clean = packed_attention(q, k, v, cut)
    k2, v2 = k.clone(), v.clone()
    k2[90:200] = value
    v2[90:200] = value
    got = packed_attention(q, k2, v2, cut)
    assert torch.equal(got[:90], clean[:90]) and torch.equal(got[200:], clean[200:])
    v3 = v.clone()
    v3[90, :, 5] = value
    got = packed_attention(q, k, v3, cut)
    keep = torch.ones(n, dtype=torch.bool, device=DEV)
    keep[5] = False
    assert torch.equal(got[:90], clean[:90]) and torch.equal(got[200:], clean[200:])
    assert torch.equal(got[:, :, keep][:128], clean[:, :, keep][:128])
    assert not bool(torch.isfinite(got[90:200, :, 5]).any())


@pytest.mark.parametrize("value", [float("nan"), -float("inf")])
@pytest.mark.parametrize("hq,hkv,n", [(16, 16, 64), (12, 12, 128), (40, 5, 64)])
def test_causal_with_two_tiles_to_an_item(hq, hkv, n, value):
    """Enough rows that the forward takes two query tiles at a time: v elements behind each of several cut points hold
    inf or NaN, inside either tile of a pair and at their border."""
    lens = [2000, 1111, 889]
    q, k, v, do, cu = _make(lens, hq, hkv, n, BF, seed=13)
    cut = torch.tensor(cu, dtype=torch.int32, device=DEV)
    clean = packed_attention(q, k, v, cut)
    tt = 128 // (hq // hkv)
    for at in (1, tt - 1, tt, tt + 1, 2 * tt, 1000, 1999):
        v2 = v.clone()
        v2[at, :, 3] = value
        got = packed_attention(q, k, v2, cut)
        assert torch.equal(got[:at], clean[:at]) and torch.equal(got[2000:], clean[2000:]), at
        assert not bool(torch.isfinite(got[at:2000, :, 3]).any()), at
        k2 = k.clone()
        k2[at:2000] = value
        got = packed_attention(q, k2, v, cut)
        assert torch.equal(got[:at], clean[:at]) and torch.equal(got[2000:], clean[2000:]), at


def test_nan_query_row_is_nan():
    q, k, v, do, cu = _make([140], 2, 1, 64, BF, seed=13)
    cut = torch.tensor(cu, dtype=torch.int32, device=DEV)
    clean = packed_attention(q, k, v, cut)
    q2 = q.clone()
    q2[33, 1, 7] = float("nan")
    got = packed_attention(q2, k, v, cut)
    assert bool(torch.isnan(got[33, 1]).all())
    rest = torch.ones(140, 2, dtype=torch.bool, device=DEV)
    rest[33, 1] = False
    assert torch.equal(got[rest], clean[rest])


@pytest.mark.parametrize("layout", ["joint", "heads_first", "odd_rows", "unaligned", "broadcast"])
def test_strides(layout):
    lens, hq, hkv, n = [100, 77], 4, 2, 64
    q, k, v, do, cu = _make(lens, hq, hkv, n, BF, seed=14, joint=False)
    total = cu[-1]
    want = _run(q, k, v, do, cu)
    if layout == "heads_first":
        q, k, v, do = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v, do))
    elif layout == "odd_rows":  # row stride not a multiple of 8: copied
        q, k, v, do = (torch.nn.functional.pad(t.reshape(total, -1), (0, 3))[:, :-3].view(t.shape) for t in (q, k, v, do))
    elif layout == "unaligned":
        q, k, v, do = (torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape) for t in (q, k, v, do))
    elif layout == "broadcast":  # both key/value heads the same memory, and a broadcast gradient
        k, v, do = k[:, :1].expand(-1, 2, -1), v[:, :1].expand(-1, 2, -1), do[:1, :1].expand(total, hq, n)
        want = _run(q, k.contiguous(), v.contiguous(), do.contiguous(), cu)
    got = _run(q, k, v, do, cu)
    for x in got:
        assert torch.equal(got[x], want[x]), x


def test_gradient_of_a_broadcast_key_is_summed():
    q, k, v, do, cu = _make([90], 4, 2, 64, BF, seed=15, joint=False)
    cut = torch.tensor(cu, dtype=torch.int32, device=DEV)
    one = k[:, :1].clone().requires_grad_(True)
    o = packed_attention(q, one.expand(-1, 2, -1), v, cut)
    (got,) = torch.autograd.grad(o, one, do)
    want = _run(q, k[:, :1].expand(-1, 2, -1), v, do, cu)["dk"]
    assert torch.equal(got, want.sum(1, keepdim=True))


def test_same_call_same_bits():
    q, k, v, do, cu = _make([1000, 300, 7, 1500], 8, 2, 128, BF, seed=16)
    a, b = _run(q, k, v, do, cu), _run(q, k, v, do, cu)
    for x in a:
        assert torch.equal(a[x], b[x]), x


@pytest.mark.parametrize("lens", [[], [0], [0, 0, 0]])
def test_nothing_to_attend(lens):
    q, k, v, do, cu = _make(lens, 4, 2, 64, BF, behind=200)
    assert all(not bool(x.any()) for x in _run(q, k, v, do, cu).values())
    q, k, v, do, cu = _make(lens, 4, 2, 64, BF, behind=0)
    assert all(x.numel() == 0 for x in _run(q, k, v, do, cu).values())


@pytest.mark.parametrize("cu", [[0, 100, 90, 200], [-1, 100, 200], [0, 100, 201], [5, 4]])
def test_row_numbers_that_do_not_rise(cu):
    q, k, v, do, _ = _make([200], 4, 2, 64, BF, seed=17)
    o = packed_attention(q, k, v, torch.tensor(cu, dtype=torch.int32, device=DEV))
    torch.cuda.synchronize()
    assert not bool(o.any())
    with pytest.raises(MeaError, match="cu_seqlens"):
        check_device_status(DEV)
    check_device_status(DEV)


def test_other_stream_and_interleaved_calls():
    q, k, v, do, cu = _make([500, 20, 333], 4, 2, 64, BF, seed=18)
    q2, k2, v2, do2, cu2 = _make([90, 1000], 4, 1, 128, BF, seed=19)
    want, want2 = _run(q, k, v, do, cu), _run(q2, k2, v2, do2, cu2)
    s, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for stream, a in ((s, (q, k, v, do, cu)), (s2, (q2, k2, v2, do2, cu2))):
            with torch.cuda.stream(stream):
                leaves = [t.detach().requires_grad_(True) for t in a[:3]]
                o = packed_attention(*leaves, torch.tensor(a[4], dtype=torch.int32, device=DEV))
                got.append((o.detach(), *torch.autograd.grad(o, leaves, a[3])))
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        for t, name in zip(x, ("o", "dq", "dk", "dv")):
            assert torch.equal(t, (want2 if i % 2 else want)[name])


def test_calls_from_other_threads():
    """The first CUDA call that a new thread makes: forward and backward (autograd's own thread) alike."""
    import threading

    q, k, v, do, cu = _make([300, 20], 4, 2, 64, BF, seed=30)
    want, got = _run(q, k, v, do, cu), {}

    def work(i):
        got[i] = _run(q, k, v, do, cu)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 3
    for x in got.values():
        assert all(torch.equal(x[n], want[n]) for n in want)


def test_captured_call_follows_the_lengths():
    """Forward and backward in a CUDA graph, replayed with other values and other lengths, two graphs in turn."""
    hq, hkv, n, total = 4, 2, 64, 400
    lens = [[400], [1, 199, 0, 200], [128, 128, 100, 0], [390, 0, 0, 3]]
    cases = [_make(x, hq, hkv, n, BF, seed=20 + i, behind=total - sum(x)) for i, x in enumerate(lens)]

    def padded(cu):
        return torch.tensor(cu + [cu[-1]] * (5 - len(cu)), dtype=torch.int32, device=DEV)

    want = [_run(*c[:4], padded(c[4]).tolist()) for c in cases]
    keep = packed_attention(*(t.detach().requires_grad_(True) for t in cases[0][:3]), padded(cases[0][4]))  # a live eager graph
    graphs = []
    for _ in range(2):
        static = [t.clone() for t in cases[0][:4]]
        cu = padded(cases[0][4]).clone()
        leaves = [t.requires_grad_(True) for t in static[:3]]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = packed_attention(*leaves, cu)
            grads = torch.autograd.grad(o, leaves, static[3])
        graphs.append((graph, static, cu, (o, *grads)))
    for i in (1, 2, 3, 0, 2):
        for graph, static, cu, out in graphs:
            with torch.no_grad():
                for a, b in zip(static, cases[i][:4]):
                    a.copy_(b)
                cu.copy_(padded(cases[i][4]))
            graph.replay()
        torch.cuda.synchronize()
        for *_, out in graphs:
            for t, name in zip(out, ("o", "dq", "dk", "dv")):
                assert torch.equal(t.detach(), want[i][name]), (i, name)
    del keep
    check_device_status(DEV)


@pytest.mark.parametrize("lens,hq,hkv", [([300, 1, 128, 2000, 77], 8, 8), ([2500], 8, 1)])
def test_backward_calls_of_one_forward_at_once(lens, hq, hkv):
    """Two captured backward calls of one kept forward, replayed on two streams at the same time, again and again: each
    draws its tiles from counters of its own."""
    q, k, v, do, cu = _make(lens, hq, hkv, 64, BF, seed=31)
    want = _run(q, k, v, do, cu)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    side = [torch.cuda.Stream() for _ in range(2)]
    cut = torch.tensor(cu, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    with torch.cuda.stream(side[0]):  # (a backward runs on its forward's stream, so that one is captured)
        o = packed_attention(*leaves, cut)
    torch.cuda.synchronize()
    graphs = []
    for s in side:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side[0]):
            grads = torch.autograd.grad(o, leaves, do, retain_graph=True)
        graphs.append((graph, s, grads))
    for _ in range(20):
        for graph, s, _g in graphs:
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for *_x, grads in graphs:
            for t, name in zip(grads, ("dq", "dk", "dv")):
                assert torch.equal(t, want[name]), name
                t.zero_()
    check_device_status(DEV)


def test_arguments_are_checked():
    q, k, v, do, cu = _make([20], 4, 2, 64, BF)
    cut = torch.tensor(cu, dtype=torch.int32, device=DEV)
    for args, err, text in (
            ((q[:, :3], k, v, cut), ValueError, "multiple"), ((q, k, v[:, :1], cut), ValueError, "k and v"),
            ((q[:10], k, v, cut), ValueError, "k and v"), ((q.float(), k.float(), v.float(), cut), TypeError, "bf16 or fp16"),
            ((q, k.half(), v, cut), TypeError, "one type"), ((q, k, v, cut.long()), TypeError, "int32"),
            ((q, k, v, cut.cpu()), ValueError, "device"), ((q[..., :60], k[..., :60], v[..., :60], cut), ValueError, "head dim"),
            ((q[0], k, v, cut), ValueError, "total"), ((q, k, v, cut, 0.0), ValueError, "scale"),
            ((q, k, v, cut[:0]), TypeError, "int32")):
        with pytest.raises(err, match=text):
            packed_attention(*args)


def test_second_derivative_is_refused():
    q, k, v, do, cu = _make([20], 2, 1, 64, BF)
    q = q.detach().requires_grad_(True)
    o = packed_attention(q, k, v, torch.tensor(cu, dtype=torch.int32, device=DEV))
    (g,) = torch.autograd.grad(o, q, do, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.float().sum(), q)
