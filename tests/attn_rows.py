"""Attention over the 8-bit cache in 64 bits with a bound of the error for every element of its own.

Row i and head h see keys j with weights w_j.  With A the largest scale * sum |q k_j| the row sees and
W = sum w_j |v_j| (a number a dim):
  scores      fp32 queries keep 22 bits of a row's largest element, bf16 ones all of theirs, and the sum over
              head_dim rounds in fp32: off by at most A (head_dim + 8) 2^-24 =: e.  A weight then moves by
              a factor of at most exp(2 e), its own change and the sum's.
  weights     held in 22 bits, exponential and scale included: 8 half steps of fp32
  sums        over n keys, 32 at a time, rescaled and joined: n / 32 + 40 half steps
which are all relative to W; what a weight loses at the bottom of its range is 2^-38 of the largest
w_j * scale_j * 127 a key.  The result is rounded once, by half a step of its type at the value; where a
power of two lies in between, by the error again."""
import math

import torch

from . import mix_ref as R


def attention(q, cache, table, lens, rows, scale, max_len):
    """out, bound [n][hq][d] in fp64; rows that see nothing have the bound 0"""
    ck, cv, ks, vs, page = cache
    n, hq, d = q.shape
    out, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    group, at = hq // ck.shape[1], R.starts(rows)
    for s, (length, r) in enumerate(zip(lens, rows)):
        m = max(0, min(length, max_len, table.shape[1] * page))
        if not m or not r:
            continue
        k, v, there = R.page_values(ck, cv, ks, vs, table[s], m, page)
        pos = torch.arange(m)
        see = there[None] & (pos[None] <= length - r + torch.arange(r)[:, None])
        keys = see.sum(-1, keepdim=True).double()
        on = table[s].long()[pos // page].clamp(0, ck.shape[0] - 1)
        for h in range(hq):
            kk, vv, qq = k[:, h // group], v[:, h // group], q[at[s]:at[s] + r, h].double()
            z = (qq @ kk.t() * scale).masked_fill(~see, -math.inf)
            w = torch.exp(z - z.amax(-1, keepdim=True).clamp(min=-1e300))
            w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
            big = (qq.abs() @ kk.abs().t() * abs(scale)).masked_fill(~see, 0.0).amax(-1, keepdim=True)
            rel = torch.expm1((2 * big * (d + 8) * R.U24).clamp(max=50.0)) + (keys / 32 + 48) * R.U24
            most = (w * vs[on, h // group].double().abs()[None]).masked_fill(~see, 0.0).amax(-1, keepdim=True)
            w = w.masked_fill(~see, 0.0)
            vv = vv.masked_fill(~there[:, None], 0.0)
            out[at[s]:at[s] + r, h] = w @ vv
            tol[at[s]:at[s] + r, h] = w @ vv.abs() * rel + most * 127 * keys * 2.0 ** -38
    return out, tol


def check(got, ref, tol, dtype, what=""):
    """|got - ref| <= half a step of `dtype` at ref + 2 tol"""
    got = got.double().cpu()
    assert got.shape == ref.shape and bool(torch.isfinite(got).all()), what + ": not finite"
    bits = {torch.bfloat16: 8, torch.float32: 24}[dtype]
    half = torch.ldexp(torch.ones_like(ref), torch.frexp(ref).exponent - 1 - bits) * (ref != 0)
    over = (got - ref).abs() - half - 2 * tol
    at = int(over.argmax())
    assert float(over.max()) <= 0, "%s: %d of %d elements off; %.9e for %.9e, bound %.3e + %.3e" % (
        what, int((over > 0).sum()), over.numel(), float(got.flatten()[at]), float(ref.flatten()[at]),
        float(half.flatten()[at]), float(2 * tol.flatten()[at]))
