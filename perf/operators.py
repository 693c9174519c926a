"""Timed cases of the packed-sequence training operators: causal attention over
packed sequences with grouped heads, layer norm, and the clipping of a list of
gradients by their global norm.

``run`` is one pass of a case: in plain torch operations where ``own`` is
False, through this package's public calls where it is True.  ``exact`` gives
the same outputs from the definitions in 64 bits.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # Causal attention forward over a packed batch of prompts.
        # A handful of short prompts, where the latency of the call counts.
        {"name": "attn_short", "op": "attn", "train": False, "dtype": "bf16", "hq": 8, "hkv": 8, "n": 64,
         "lens": "1,17,128,3,64,90,5", "pad": 0},
        # A ragged batch with four query heads to a key/value head.
        {"name": "attn_prompts", "op": "attn", "train": False, "dtype": "bf16", "hq": 16, "hkv": 4, "n": 128,
         "lens": "2048,1531,700,1999,64,1,1200,333", "pad": 0},
        # One long prompt at the long-context block's length and heads.
        {"name": "attn_long", "op": "attn", "train": False, "dtype": "bf16", "hq": 16, "hkv": 2, "n": 128,
         "lens": "16384", "pad": 0},
        # Forward and backward.  A small packed batch in half precision.
        {"name": "attn_train_short", "op": "attn", "train": True, "dtype": "fp16", "hq": 8, "hkv": 8, "n": 64,
         "lens": "256,100,1,400,77,190", "pad": 0},
        # Documents of up to 2048 tokens packed into one row at the 50M block's heads, with padding behind them.
        {"name": "attn_train_docs", "op": "attn", "train": True, "dtype": "bf16", "hq": 8, "hkv": 8, "n": 64,
         "lens": "2048,2048,1777,1024,1500,311,2048,640,999,2001,1310,57,820,2048,1903,733", "pad": 113},
        # Two long documents with grouped heads.
        {"name": "attn_train_long", "op": "attn", "train": True, "dtype": "bf16", "hq": 16, "hkv": 4, "n": 128,
         "lens": "12289,4095", "pad": 0},
        # Layer norm forward and backward: a few rows (latency), the long-context block's rows and width, and an odd
        # width in single precision.
        {"name": "norm_short", "op": "norm", "train": True, "dtype": "bf16", "rows": 64, "c": 512, "bias": True},
        {"name": "norm_train", "op": "norm", "train": True, "dtype": "bf16", "rows": 65536, "c": 2048, "bias": True},
        {"name": "norm_odd", "op": "norm", "train": True, "dtype": "fp32", "rows": 10007, "c": 1001, "bias": False},
        # Clipping by the global norm: the five weights of the 50M block, a twelve-layer model of blocks and 4C MLPs,
        # and a smaller one with fp32 gradients.
        {"name": "clip_block", "op": "clip", "dtype": "bf16", "c": 512, "layers": 1, "mlp": False, "max_norm": 1.0},
        {"name": "clip_model", "op": "clip", "dtype": "bf16", "c": 2048, "layers": 12, "mlp": True, "max_norm": 1.0},
        {"name": "clip_fp32", "op": "clip", "dtype": "fp32", "c": 1024, "layers": 14, "mlp": True, "max_norm": 0.5},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn_train", "attn_train", "norm", "norm", "clip"])
    if op.startswith("attn"):
        hkv = rng.choice([1, 2, 3, 4, 8])
        hq = hkv * rng.choice([g for g in (1, 2, 3, 4, 6, 7, 8) if g * hkv <= 24])
        total, seqs = _log_int(rng, 8, 16384), _log_int(rng, 1, 64)
        shares = [rng.expovariate(1.0) + 0.05 for _ in range(seqs)]
        lens = [max(1, int(total * s / sum(shares))) for s in shares]
        while len(lens) * hq * max(lens) ** 2 > 1.2e9:  # what the padded plain form holds
            lens[lens.index(max(lens))] //= 2
        if rng.random() < 0.3:
            lens.insert(rng.randrange(len(lens) + 1), 0)
        return {"op": "attn", "train": op == "attn_train", "dtype": rng.choice(["bf16", "bf16", "fp16"]), "hq": hq,
                "hkv": hkv, "n": rng.choice([32, 40, 64, 64, 80, 96, 128, 128]),
                "lens": ",".join(str(x) for x in lens), "pad": rng.choice([0, 0, rng.randrange(1, 200)])}
    if op == "norm":
        c = _log_int(rng, 16, 16384)
        if rng.random() < 0.6:
            c = max(16, c // 64 * 64)
        rows = _log_int(rng, 1, min(65536, (65536 * 2048) // c))
        return {"op": "norm", "train": rng.random() < 0.8, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                "rows": rows, "c": c, "bias": rng.random() < 0.6}
    c = 8 * _log_int(rng, 4, 192)
    return {"op": "clip", "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "c": c,
            "layers": rng.randrange(1, 13), "mlp": rng.random() < 0.6, "max_norm": rng.choice([0.5, 1.0, 2.0])}


# -- inputs ----------------------------------------------------------------------------------------------------------
def _cu(lens):
    cu = [0]
    for x in lens:
        cu.append(cu[-1] + x)
    return cu


def _clip_shapes(case):
    c, shapes = case["c"], []
    for _ in range(case["layers"]):
        shapes += [(c, c)] * 5 + [(c,), (c,)]
        if case["mlp"]:
            shapes += [(4 * c, c), (c, 4 * c)]
    return shapes


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def randn(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    if case["op"] == "attn":
        lens = [int(x) for x in case["lens"].split(",")]
        hq, hkv, n, total = case["hq"], case["hkv"], case["n"], sum(lens) + case["pad"]
        # q, k and v as a joint projection leaves them: views of one [total, (hq + 2 hkv) n] tensor
        joint = randn(total, hq + 2 * hkv, n)
        q, k, v = (t.detach().requires_grad_(case["train"]) for t in joint.split([hq, hkv, hkv], dim=1))
        s = {"q": q, "k": k, "v": v, "cu": torch.tensor(_cu(lens), dtype=torch.int32, device="cuda"),
             "longest": max(lens)}
        if case["train"]:
            s["do"] = randn(total, hq, n)
    elif case["op"] == "norm":
        rows, c = case["rows"], case["c"]
        # a residual stream: rows of different size, off centre
        x = (randn(rows, c, dtype=torch.float32) * (0.5 + torch.rand(rows, 1, generator=g, device="cuda"))
             + 0.3 * randn(rows, 1, dtype=torch.float32)).to(dt)
        s = {"x": x.requires_grad_(case["train"]),
             "w": (1.0 + 0.1 * randn(c, dtype=torch.float32)).to(dt).requires_grad_(case["train"]),
             "b": (0.1 * randn(c, dtype=torch.float32)).to(dt).requires_grad_(case["train"]) if case["bias"] else None,
             "eps": 1e-5}
        if case["train"]:
            s["dy"] = randn(rows, c)
    else:
        shapes = _clip_shapes(case)
        at, end = [], 0
        for shape in shapes:  # every gradient a view of one flat buffer, 8-element aligned
            at.append(end)
            end += (math.prod(shape) + 7) // 8 * 8
        flat = torch.zeros(end, device="cuda", dtype=dt)
        params = []
        for shape, o in zip(shapes, at):
            view = flat[o:o + math.prod(shape)].view(shape)
            view.copy_(0.01 * randn(*shape, dtype=torch.float32))
            p = torch.nn.Parameter(torch.zeros(shape, device="cuda", dtype=dt))
            p.grad = view
            params.append(p)
        s = {"params": params, "flat": flat, "max_norm": case["max_norm"]}
    return {"case": dict(case), **s}


# -- one pass ----------------------------------------------------------------------------------------------------------
def _plain_attn(s):
    """Sequences padded to the longest one: scores, softmax and products in fp32, and their gradients by the formula.
    A padded key comes after every real query, so the causal mask covers it; padded rows are dropped at the end."""
    q, k, v, cu, longest = s["q"], s["k"], s["v"], s["cu"].long(), s["longest"]
    (total, hq, n), hkv, dt = q.shape, k.shape[1], q.dtype
    group, seqs = hq // hkv, cu.numel() - 1
    pos = torch.arange(longest, device=q.device)
    at = torch.where(pos < (cu[1:] - cu[:-1])[:, None], cu[:-1, None] + pos, total)

    def padded(t, g):  # [total, heads, n] -> [seqs, hkv, g * longest, n] in fp32
        t = torch.cat([t.float(), t.new_zeros(1, t.shape[1], n, dtype=torch.float32)])[at]
        return t.view(seqs, longest, hkv, g, n).permute(0, 2, 3, 1, 4).reshape(seqs, hkv, g * longest, n)

    def packed(t, g):
        out = t.new_zeros(total + 1, hkv * g, n)
        out[at] = t.view(seqs, hkv, g, longest, n).permute(0, 3, 1, 2, 4).reshape(seqs, longest, hkv * g, n)
        out[total] = 0
        return out[:total].to(dt)

    qp, kp, vp = padded(q, group), padded(k, 1), padded(v, 1)
    scale = n ** -0.5
    p = torch.matmul(qp, kp.transpose(-1, -2)).mul_(scale)
    p.view(seqs, hkv, group, longest, longest).masked_fill_(pos[None, :] > pos[:, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    p.div_(p.sum(-1, keepdim=True))
    op = torch.matmul(p, vp)
    out = {"o": packed(op, group)}
    if "do" in s:
        dop = padded(s["do"], group)
        out["dv"] = packed(torch.matmul(p.transpose(-1, -2), dop), 1)
        ds = torch.matmul(dop, vp.transpose(-1, -2)).sub_((dop * op).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        out["dq"] = packed(torch.matmul(ds, kp), group)
        out["dk"] = packed(torch.matmul(ds.transpose(-1, -2), qp), 1)
    return out


def _plain_norm(s):
    x, w, dt = s["x"].float(), s["w"].float(), s["x"].dtype
    mean = x.mean(-1, keepdim=True)
    xc = x - mean
    rstd = torch.rsqrt((xc * xc).mean(-1, keepdim=True) + s["eps"])
    xhat = xc * rstd
    y = xhat * w
    if s["b"] is not None:
        y = y + s["b"].float()
    out = {"y": y.to(dt)}
    if "dy" in s:
        dy = s["dy"].float()
        g = dy * w
        dx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
        out["dx"], out["dw"] = dx.to(dt), (dy * xhat).sum(0).to(dt)
        if s["b"] is not None:
            out["db"] = dy.sum(0).to(dt)
    return out


def _plain_clip(s, max_norm):
    g = s["flat"].float()
    norm = (g * g).sum().sqrt()
    s["flat"].copy_(g * (max_norm / (norm + 1e-6)).clamp(max=1.0))
    return {"norm": norm, "grads": s["flat"]}


def run(s):
    op = s["case"]["op"]
    if op == "clip":
        # The threshold falls by 1e-5 a pass, so that every pass scales, as with new gradients every step.
        max_norm, s["max_norm"] = s["max_norm"], s["max_norm"] * (1 - 1e-5)
        if own:
            from memory_efficient_attn_layer_b200 import clip_grad_norm_
            return {"norm": clip_grad_norm_(s["params"], max_norm), "grads": s["flat"]}
        with torch.no_grad():
            return _plain_clip(s, max_norm)
    if not own:
        with torch.no_grad():
            return _plain_attn(s) if op == "attn" else _plain_norm(s)
    if op == "attn":
        from memory_efficient_attn_layer_b200 import packed_attention
        o = packed_attention(s["q"], s["k"], s["v"], s["cu"])
        if "do" not in s:
            return {"o": o}
        dq, dk, dv = torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])
        return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}
    from memory_efficient_attn_layer_b200 import layer_norm
    y = layer_norm(s["x"], s["w"], s["b"], s["eps"])
    if "dy" not in s:
        return {"y": y}
    leaves = [t for t in (s["x"], s["w"], s["b"]) if t is not None]
    grads = torch.autograd.grad(y, leaves, s["dy"])
    return {"y": y.detach(), **dict(zip(("dx", "dw", "db"), grads))}


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "attn":
        lens = [int(x) for x in case["lens"].split(",")]
        rows, n = sum(lens) + case["pad"], case["n"]
        pairs = sum(x * (x + 1) // 2 for x in lens)
        qo, kv = rows * case["hq"] * n * size, rows * case["hkv"] * n * size
        if not case["train"]:
            return {"bytes": 2 * qo + 2 * kv, "flops": 4 * pairs * case["hq"] * n}
        return {"bytes": 4 * qo + 4 * kv, "flops": 14 * pairs * case["hq"] * n}  # 2 products forward, 5 backward
    if case["op"] == "norm":
        m = case["rows"] * case["c"]
        vec = case["c"] * (2 if case["bias"] else 1)
        if not case["train"]:
            return {"bytes": (2 * m + vec) * size, "flops": 8 * m}
        return {"bytes": (4 * m + 2 * vec) * size, "flops": 20 * m}
    m = sum(math.prod(x) for x in _clip_shapes(case))
    return {"bytes": 2 * m * size, "flops": 3 * m}


# -- the definitions in 64 bits ------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "attn":
            return _exact_attn(s)
        if case["op"] == "norm":
            return _exact_norm(s)
        g = s["flat"].double()
        norm = torch.linalg.vector_norm(g)
        return {"norm": norm, "grads": g * min(1.0, s["max_norm"] / (float(norm) + 1e-6))}


def _exact_attn(s):
    """One head of one sequence at a time, in blocks of query rows."""
    q, k, v, train = s["q"], s["k"], s["v"], "do" in s
    group, scale = q.shape[1] // k.shape[1], 1.0 / math.sqrt(q.shape[2])
    o, dq = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    dk, dv = (torch.zeros(k.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    ends = s["cu"].tolist()
    for lo, hi in zip(ends, ends[1:]):
        for h in range(q.shape[1] if hi > lo else 0):
            j = h // group
            kk, vv = k[lo:hi, j].double(), v[lo:hi, j].double()
            for a in range(lo, hi, 4096):
                b = min(a + 4096, hi)
                keys = slice(0, b - lo)
                qq = q[a:b, h].double()
                score = scale * (qq @ kk[keys].T)
                seen = torch.arange(b - lo, device=q.device)[None, :] <= torch.arange(a - lo, b - lo, device=q.device)[:, None]
                lse = torch.logsumexp(torch.where(seen, score, -math.inf), 1, keepdim=True)
                p = torch.where(seen, torch.exp(score - lse), 0.0)
                o[a:b, h] = p @ vv[keys]
                if train:
                    do = s["do"][a:b, h].double()
                    dp = do @ vv[keys].T
                    ds = p * (dp - (p * dp).sum(1, keepdim=True))
                    dq[a:b, h] = scale * (ds @ kk[keys])
                    dk[lo:b, j] += scale * (ds.T @ qq)
                    dv[lo:b, j] += p.T @ do
    return {"o": o, "dq": dq, "dk": dk, "dv": dv} if train else {"o": o}


def _exact_norm(s):
    x, w = s["x"].double(), s["w"].double()
    var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
    sd = torch.sqrt(var + s["eps"])
    z = (x - mean) / sd
    out = {"y": z * w + (0.0 if s["b"] is None else s["b"].double())}
    if "dy" in s:
        dy, c = s["dy"].double(), x.shape[1]
        gw = dy * w
        out["dx"] = (c * gw - gw.sum(1, keepdim=True) - z * (gw * z).sum(1, keepdim=True)) / (c * sd)
        out["dw"] = torch.einsum("rc,rc->c", dy, z)
        if s["b"] is not None:
            out["db"] = dy.sum(0)
    return out
