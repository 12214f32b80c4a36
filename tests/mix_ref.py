"""Plain 64-bit forms of the token mixers, the 8-bit cache and the log probabilities (CPU), and the
small helpers their GPU tests share."""
import math

import numpy as np
import torch

U24 = 2.0 ** -24          # half a step of fp32, relative
U_BF16 = 2.0 ** -8        # half a step of bf16, relative


def starts(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def gated_delta(q, k, v, g, beta, state, lens, scale, l2norm):
    """q, k [n][hk][dk], v [n][hv][dv], g, beta [n][hv], state [seqs][hv][dv][dk]: the recurrence,
    token by token in fp64.  Returns out [n][hv][dv] and the final states."""
    q, k, v, g, beta, S = (t.double() for t in (q, k, v, g, beta, state))
    S = S.clone()
    if l2norm:
        q = q / (q.square().sum(-1, keepdim=True) + 1e-6).sqrt()
        k = k / (k.square().sum(-1, keepdim=True) + 1e-6).sqrt()
    rep = v.shape[1] // q.shape[1]
    q, k = q.repeat_interleave(rep, 1), k.repeat_interleave(rep, 1)
    out = torch.zeros_like(v)
    at = starts(lens)
    for s, n in enumerate(lens):
        for t in range(at[s], at[s] + n):
            st = S[s] * g[t].exp()[:, None, None]
            u = beta[t][:, None] * (v[t] - (st * k[t][:, None, :]).sum(-1))
            st = st + u[:, :, None] * k[t][:, None, :]
            out[t] = scale * (st * q[t][:, None, :]).sum(-1)
            S[s] = st
    return out, S


def page_values(codes_k, codes_v, ks, vs, table_row, n, page):
    """Keys, values [n][heads][dim] of one sequence and which of its tokens are there."""
    heads, dim = codes_k.shape[1], codes_k.shape[3]
    k = torch.zeros(n, heads, dim, dtype=torch.float64)
    v = torch.zeros_like(k)
    there = torch.zeros(n, dtype=torch.bool)
    for p0 in range(0, n, page):
        at = p0 // page
        p = int(table_row[at]) if at < len(table_row) else -1
        if 0 <= p < codes_k.shape[0]:
            m = min(page, n - p0)
            k[p0:p0 + m] = codes_k[p, :, :m].double().transpose(0, 1) * ks[p].double()[None, :, None]
            v[p0:p0 + m] = codes_v[p, :, :, :m].double().permute(2, 0, 1) * vs[p].double()[None, :, None]
            there[p0:p0 + m] = True
    return k, v, there


def attention(q, cache, table, lens, rows, scale, max_len):
    """q [n][hq][d]; cache = (k codes, v codes, k scales, v scales, page_tokens).  fp64.  Also gives
    the largest scale * sum |q_i k_i| of a visible pair and the largest |v|."""
    ck, cv, ks, vs, page = cache
    out = torch.zeros(q.shape, dtype=torch.float64)
    at, most, vmax = starts(rows), 0.0, 0.0
    group = q.shape[1] // ck.shape[1]
    for s, (n, r) in enumerate(zip(lens, rows)):
        m = max(0, min(n, max_len, table.shape[1] * page))
        k, v, there = page_values(ck, cv, ks, vs, table[s], m, page)
        for i in range(r):
            see = there & (torch.arange(m) <= n - r + i)
            if not see.any():
                continue
            for h in range(q.shape[1]):
                kk, vv, qq = k[see][:, h // group], v[see][:, h // group], q[at[s] + i, h].double()
                z = kk @ qq * scale
                most = max(most, float((kk.abs() @ qq.abs()).max()) * abs(scale))
                vmax = max(vmax, float(vv.abs().max()))
                out[at[s] + i, h] = torch.softmax(z, 0) @ vv
    return out, most, vmax


def append(cache, table, lens, rows, k, v):
    """Writes rows into copies of the cache's tensors: (k codes, v codes, k scales, v scales)."""
    ck, cv, ks, vs, page = cache
    ck, cv, ks, vs = ck.clone(), cv.clone(), ks.clone(), vs.clone()
    at = starts(rows)
    for s, (n, r) in enumerate(zip(lens, rows)):
        pos = max(0, n - r)
        while pos < n:
            col = pos // page
            take = min(page - pos % page, n - pos)
            p = int(table[s, col]) if col < table.shape[1] else -1
            if 0 <= p < ck.shape[0]:
                keep = pos % page
                row = at[s] + r - n + pos
                for x, codes, sc in ((k, ck[p], ks), (v, cv[p].transpose(1, 2), vs)):
                    x = x[row:row + take].double()                       # [take][heads][dim]
                    fin = torch.where(torch.isfinite(x), x.abs(), 0.0)
                    amax = fin.amax((0, 2)).float().numpy()
                    new = torch.from_numpy((amax * (np.float32(1) / np.float32(127))).astype(np.float32))
                    old = sc[p].clone() if keep else torch.zeros_like(new)
                    new = torch.maximum(old, new)
                    div = new.double()[:, None, None]
                    if keep:
                        again = torch.where(div > 0, torch.round(codes[:, :keep].double() * old.double()[:, None, None] / div), 0.0)
                        codes[:, :keep] = torch.where((new != old)[:, None, None], again, codes[:, :keep].double()).to(torch.int8)
                    xt = x.transpose(0, 1)
                    qn = torch.where(div > 0, torch.round(xt / div), torch.where(torch.isinf(xt), xt, 0.0))
                    qn = torch.where(torch.isnan(xt), 0.0, qn).clamp(-127, 127)
                    codes[:, keep:keep + take] = qn.to(torch.int8)
                    sc[p] = new
            pos += take
    return ck, cv, ks, vs


def logprobs(x, tokens, top_n):
    """x [rows][vocab] fp32 without NaN / +inf."""
    x = x.double()
    rows, vocab = x.shape
    lp = torch.full((rows,), -math.inf, dtype=torch.float64)
    ent = torch.zeros(rows, dtype=torch.float64)
    ids = torch.zeros(rows, top_n, dtype=torch.int32)
    top = torch.zeros(rows, top_n, dtype=torch.float64)
    for r in range(rows):
        none = bool((x[r] == -math.inf).all())
        p = torch.full_like(x[r], -math.inf)
        if not none:
            # (the maximum's own 1 apart: log(1 + z) of a tiny z keeps its digits)
            m, first = x[r].max(0)
            d = x[r] - m
            e = d.exp()
            e[first] = 0.0
            log_z = torch.log1p(e.sum())
            p = d - log_z
            ent[r] = log_z - torch.where(e > 0, e * d, 0.0).sum() / (1 + e.sum())
        t = int(tokens[r])
        if 0 <= t < vocab:
            lp[r] = p[t]
        order = np.lexsort((np.arange(vocab), -x[r].numpy()))[:top_n]
        ids[r] = torch.from_numpy(order.astype(np.int32))
        top[r] = p[torch.from_numpy(order.copy())]
    return lp, ent, ids, top


def close(got, ref, tol_abs, tol_rel=0.0, what=""):
    """Elementwise |got - ref| <= tol_abs + tol_rel |ref|."""
    got, ref = got.double().cpu(), ref.double().cpu()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert bool(torch.isfinite(got).all()), what + ": not finite"
    over = ((got - ref).abs() - (tol_abs + tol_rel * ref.abs())).max() if got.numel() else torch.tensor(0.0)
    assert float(over) <= 0, "%s: off by %.3e more than %.3e + %.1e |ref|; largest error %.3e of %.3e" % (
        what, float(over), tol_abs, tol_rel, float((got - ref).abs().max()), float(ref.abs().max()))
