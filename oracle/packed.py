"""Packed causal attention in fp64, with bounds on what a 16-bit kernel may differ by.

``attention`` evaluates o, dq, dk, dv from the definition, one sequence and
head at a time.  With ``eps`` it also returns, element by element, how far a
kernel may be off that rounds P, dS, o and the gradients to a type of that
``torch.finfo(t).eps`` (half a step u = eps / 2 each) and works in fp32
otherwise:

* P carries e = 3e-4 on top of its rounding: the polynomial exponential
  (8.4e-5), and the fp32 score and log-sum-exp, whose absolute errors (a few
  2^-24 times scores of up to about 60) the exponential turns into relative ones.
* o_id: (u + e) sum_j p_ij |v_jd| + u |o_id|.
* dv_jd: (u + e) sum_i p_ij |do_id| + u |dv_jd|.
* delta_i is formed from the rounded o: off by D_i = sum_d |do_id| (bound of o_id)
  plus its own fp32 sum.
* dS_ij: (u + e) |dS_ij| + p_ij (D_i + fp32 sums of dP), so dq and dk: that
  against |k|, |q|, plus u of the result.
* ``tiny`` is the absolute spacing below which the type's values cannot follow
  (half of fp16's smallest subnormal; 0 for bf16): it adds tiny times the sum of
  the other operand's magnitudes.
"""
import math

import torch

E = 3e-4
F32 = 2.0 ** -22  # fp32 sums of up to 128 products and sums over keys: a few half steps


def attention(q, k, v, cu, scale=None, do=None, eps=None, tiny=0.0):
    """{"o", "dq", "dk", "dv"} in fp64 and, with eps, {"bo", "bdq", "bdk", "bdv"}."""
    total, hq, n = q.shape
    group = hq // k.shape[1]
    scale = 1.0 / math.sqrt(n) if scale is None else scale
    q, k, v = q.double(), k.double(), v.double()
    do = None if do is None else do.double()
    names = ["o"] + (["dq", "dk", "dv"] if do is not None else [])
    like = {"o": q, "dq": q, "dk": k, "dv": k}
    out = {x: torch.zeros_like(like[x]) for x in names}
    if eps is not None:
        out.update({"b" + x: torch.zeros_like(like[x]) for x in names})
        u = eps / 2
    for lo, hi in zip(cu, cu[1:]):
        if hi <= lo:
            continue
        seen = torch.ones(hi - lo, hi - lo, dtype=torch.bool, device=q.device).tril()
        for h in range(hq):
            g = h // group
            Q, K, V = q[lo:hi, h], k[lo:hi, g], v[lo:hi, g]
            p = torch.softmax((scale * (Q @ K.T)).masked_fill(~seen, -math.inf), dim=1)
            o = p @ V
            out["o"][lo:hi, h] = o
            if eps is not None:
                bo = (u + E) * (p @ V.abs()) * (1 + u) + u * o.abs() + tiny * (seen.double() @ V.abs() + 1)
                out["bo"][lo:hi, h] = bo
            if do is None:
                continue
            D = do[lo:hi, h]
            dp = D @ V.T
            ds = p * (dp - (D * o).sum(1, keepdim=True))
            out["dv"][lo:hi, g] += p.T @ D
            out["dq"][lo:hi, h] = scale * (ds @ K)
            out["dk"][lo:hi, g] += scale * (ds.T @ Q)
            if eps is not None:
                off = (D.abs() * bo).sum(1, keepdim=True) + F32 * (D.abs() * o.abs()).sum(1, keepdim=True)
                bds = (u + E) * ds.abs() + p * (off + F32 * (D.abs() @ V.abs().T)) + tiny * seen.double()
                out["bdv"][lo:hi, g] += (u + E) * (p.T @ D.abs()) + tiny * (seen.double().T @ D.abs())
                out["bdq"][lo:hi, h] = scale * (bds @ K.abs())
                out["bdk"][lo:hi, g] += scale * (bds.T @ Q.abs())
    if eps is not None and do is not None:
        for x in ("dq", "dk", "dv"):
            out["b" + x] = out["b" + x] * (1 + u) + u * out[x].abs() + tiny
    return out
