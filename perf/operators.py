"""Cases of the token mixers, the 8-bit cache and the log probabilities, with their plain forms.

`own` selects what run() does: False computes the operator with elementary torch operations in
32 bits (64 where a value sits next to a rounding border), True makes the calls a user of the
framework makes.  One case is one call (the cache write is a write and the read-back of what it
stored).

  gdn       gated delta rule: state [v_dim][k_dim] a value head, one token per sequence or a chunk
  attn      attention over the paged 8-bit cache: one row per sequence or a chunk of new rows
  append    rows written into the cache, block scales updated; the stored values are returned
  logprobs  log probability of a given token, entropy and top alternatives of rows of logits
"""
import math

import torch

own = False

BF16, F32 = "bf16", "f32"
VOCAB = 248320


def _dt(case):
    return torch.bfloat16 if case["dtype"] == BF16 else torch.float32


# ------------------------------------------------------------------------------------------ cases
def listed():
    # head layouts: 16 key / 32 value heads of 128 are the ones the GatedDeltaNet projections of
    # this repository produce (2048 -> 2048 + 2048 + 4096 + 4096)
    gdn = {"op": "gdn", "k_heads": 16, "v_heads": 32, "k_dim": 128, "v_dim": 128}
    attn = {"op": "attn", "q_heads": 16, "kv_heads": 2, "head_dim": 256, "page": 64}
    return [
        # one sequence generating: the call's latency
        dict(gdn, name="gdn step 1 seq", dtype=F32, lens="1"),
        # a serving batch generating: the states' traffic
        dict(gdn, name="gdn step 48 seqs", dtype=BF16, lens=",".join(["1"] * 48)),
        # a short prompt, ends inside a chunk
        dict(gdn, name="gdn prompt 77", dtype=F32, lens="77"),
        # three prompts of one batch, one of them a single token, ragged ends
        dict(gdn, name="gdn ragged batch", dtype=BF16, lens="512,1,1203"),
        # a long prompt of one sequence: the serial chain over chunks counts
        dict(gdn, name="gdn prompt 8192", dtype=F32, lens="8192"),
        # one sequence generating on a short context: latency
        dict(attn, name="attn step 1 seq", dtype=F32, rows="1", ctx="999"),
        # a serving batch generating on ragged contexts: the cache's traffic
        dict(attn, name="attn step 32 seqs", dtype=BF16, rows=",".join(["1"] * 32),
             ctx=",".join(str(500 + 503 * i) for i in range(32))),
        # two short prompts, narrower heads, pages that end inside a tile
        dict(attn, name="attn prompt ragged", dtype=F32, rows="129,300", ctx="129,300", q_heads=8, kv_heads=2,
             head_dim=128, page=16),
        # a chunk of a long prompt behind what the cache holds
        dict(attn, name="attn chunk 2048", dtype=BF16, rows="2048", ctx="8192"),
        # a prompt's rows into the cache, first page partly filled
        dict(op="append", name="append prompt 1500", kv_heads=2, head_dim=256, page=64, dtype=F32, rows="1500",
             ctx="1530"),
        # log probability of one generated token
        dict(op="logprobs", name="logprobs 1 row", rows=1, vocab=VOCAB, top=20),
        # scoring a prompt
        dict(op="logprobs", name="logprobs 257 rows", rows=257, vocab=VOCAB, top=5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["gdn", "gdn", "attn", "attn", "append", "logprobs"])
    dtype = rng.choice([BF16, F32])
    if op == "gdn":
        k_heads = rng.choice([1, 2, 4, 8, 16])
        v_heads = k_heads * rng.choice([1, 2, 3])
        k_dim, v_dim = rng.choice([64, 128]), rng.choice([64, 80, 128, 256])
        if rng.random() < 0.4:
            lens = [1] * _log(rng, 1, 48)
        else:
            lens = [_log(rng, 1, 4000) for _ in range(rng.choice([1, 1, 2, 3, 5]))]
        while sum(lens) * v_heads * v_dim > 8192 * 32 * 128 or max(lens) * len(lens) > 16384:
            lens.pop()
        return {"op": op, "k_heads": k_heads, "v_heads": v_heads, "k_dim": k_dim, "v_dim": v_dim, "dtype": dtype,
                "lens": ",".join(map(str, lens))}
    if op == "attn":
        kv = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 2, 3, 4, 8, 16])
        d, page = rng.choice([64, 128, 256]), rng.choice([16, 32, 64, 128])
        if rng.random() < 0.5:
            n = _log(rng, 1, 32)
            rows, ctx = [1] * n, [_log(rng, 1, 30000) for _ in range(n)]
        else:
            n = rng.choice([1, 1, 2, 3])
            rows = [_log(rng, 2, 2000) for _ in range(n)]
            ctx = [r + rng.choice([0, _log(rng, 1, 6000)]) for r in rows]
        # no more scores or cache than the largest listed cases
        while (len(rows) * max(rows) * max(ctx) * kv * group > 2048 * 8192 * 16
               or sum(ctx) * kv * d > 32 * 8300 * 2 * 256 or len(rows) * max(ctx) * kv * d > 32 * 16384 * 2 * 256):
            if len(rows) > 1:
                rows.pop()
                ctx.pop()
            else:
                ctx[0] = max(rows[0], ctx[0] // 2)
                kv = max(1, kv // 2)
        return {"op": op, "q_heads": kv * group, "kv_heads": kv, "head_dim": d, "page": page, "dtype": dtype,
                "rows": ",".join(map(str, rows)), "ctx": ",".join(map(str, ctx))}
    if op == "append":
        rows = [_log(rng, 1, 500) for _ in range(rng.choice([1, 2, 3]))]
        return {"op": op, "kv_heads": rng.choice([1, 2, 4]), "head_dim": rng.choice([64, 128, 256]),
                "page": rng.choice([16, 32, 64, 128]), "dtype": dtype, "rows": ",".join(map(str, rows)),
                "ctx": ",".join(str(r + rng.choice([0, rng.randrange(200)])) for r in rows)}
    return {"op": op, "rows": _log(rng, 1, 257), "vocab": _log(rng, 1000, VOCAB), "top": rng.choice([0, 1, 5, 20, 32])}


def _ints(text):
    return [int(v) for v in text.split(",")]


# --------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _starts(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def prepare(case, seed):
    g = _gen(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def rand(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    if case["op"] == "gdn":
        return _prepare_gdn(case, randn, rand)
    if case["op"] == "logprobs":
        logits = randn(case["rows"], case["vocab"]) * 2.5
        # a few tokens carry most of the probability, as a trained model's rows do
        at = torch.randint(0, case["vocab"], (case["rows"], 8), generator=g, device="cuda")
        logits.scatter_add_(1, at, 4.0 + 8.0 * rand(case["rows"], 8))
        tokens = at[:, 0].to(torch.int32).contiguous()
        n = case["top"]
        return {"case": case, "logits": logits, "tokens": tokens,
                "logprob": torch.empty(case["rows"], device="cuda"), "entropy": torch.empty(case["rows"], device="cuda"),
                "ids": torch.empty(case["rows"], n, dtype=torch.int32, device="cuda"),
                "top": torch.empty(case["rows"], n, device="cuda")}
    return _prepare_cache(case, g, randn, rand)


def _prepare_gdn(case, randn, rand):
    hk, hv, dk, dv, dt = case["k_heads"], case["v_heads"], case["k_dim"], case["v_dim"], _dt(case)
    lens = _ints(case["lens"])
    n = sum(lens)
    # q | k | v of a token lie in one row, as the projection and the convolution leave them
    qkv = torch.nn.functional.silu(randn(n, 2 * hk * dk + hv * dv)).to(dt)
    # decay of a token and head: -exp(A) softplus(a), A a head's parameter
    a_head = torch.log(1.0 + 15.0 * rand(hv))
    decay = -torch.exp(a_head) * torch.nn.functional.softplus(randn(n, hv) - 4.0)
    beta = torch.sigmoid(randn(n, hv))
    state = 0.1 * randn(len(lens), hv, dv, dk)
    return {"case": case, "lens": lens, "qkv": qkv, "g": decay.contiguous(), "beta": beta.contiguous(),
            "state": state, "new_state": torch.empty_like(state),
            "out": torch.empty(n, hv, dv, dtype=dt, device="cuda"), "scale": dk ** -0.5}


def _prepare_cache(case, g, randn, rand):
    kv, d, page, dt = case["kv_heads"], case["head_dim"], case["page"], _dt(case)
    rows, ctx = _ints(case["rows"]), _ints(case["ctx"])
    per_seq = [-(-c // page) for c in ctx]
    n_pages, max_pages = sum(per_seq) + 3, max(per_seq)
    # a sequence's pages lie anywhere in the pool; table entries behind the last page are -1
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    slot = torch.arange(max_pages, device="cuda")[None, :]
    first = torch.tensor(_starts(per_seq)[:-1], device="cuda")[:, None]
    have = torch.tensor(per_seq, device="cuda")[:, None]
    table = torch.where(slot < have, order[(first + slot).clamp(max=n_pages - 1)], torch.full_like(slot, -1, dtype=torch.int32))

    def codes(*shape):
        return (randn(*shape) * 36.0).clamp_(-127, 127).round_().to(torch.int8)

    s = {"case": case, "rows": rows, "ctx": ctx, "pages": table.to(torch.int32).contiguous(), "n_pages": n_pages,
         "len": torch.tensor(ctx, dtype=torch.int32, device="cuda"),
         "k": codes(n_pages, kv, page, d), "v": codes(n_pages, kv, d, page),
         "k_scale": 0.01 + 0.02 * rand(n_pages, kv), "v_scale": 0.01 + 0.02 * rand(n_pages, kv)}
    n = sum(rows)
    if case["op"] == "attn":
        s["q"] = (randn(n, case["q_heads"], d) * 2.5).to(dt)
        s["scale"] = d ** -0.5
        s["out"] = torch.empty_like(s["q"])
    else:
        s["new_k"] = (randn(n, kv, d) * (0.5 + 2.0 * rand(n, kv, 1))).to(dt)
        s["new_v"] = (randn(n, kv, d) * (0.5 + rand(n, kv, 1))).to(dt)
        # what is read back: the new rows and what their first page held already
        s["back"] = [r + (c - r) % page for r, c in zip(rows, ctx)]
        s["k_out"] = torch.empty(sum(s["back"]), kv, d, device="cuda")
        s["v_out"] = torch.empty_like(s["k_out"])
    return s


# ------------------------------------------------------------------------------------------ runs
def run(state):
    if own:
        return {"gdn": _own_gdn, "attn": _own_attn, "append": _own_append, "logprobs": _own_logprobs}[state["case"]["op"]](state)
    return {"gdn": _plain_gdn, "attn": _plain_attn, "append": _plain_append,
            "logprobs": _plain_logprobs}[state["case"]["op"]](state)


# the framework's calls: a context and, per state, the descriptors over its buffers
_context = []


def _ctx():
    if not _context:
        from finchmoe_amd import FinchHip
        _context.append(FinchHip(0))
    return _context[0]


def _code(case):
    from finchmoe_amd import binding
    return binding.DTYPE_BF16 if case["dtype"] == BF16 else binding.DTYPE_F32


def _own_gdn(s):
    ctx = _ctx()
    if "plan" not in s:
        c, qkv = s["case"], s["qkv"]
        kw = c["k_heads"] * c["k_dim"]
        at, size = qkv.data_ptr(), qkv.element_size()
        n = len(s["lens"])
        s["plan"] = ctx.gated_delta_args(
            n_seq=n, k_heads=c["k_heads"], v_heads=c["v_heads"], k_dim=c["k_dim"], v_dim=c["v_dim"],
            dtype=_code(c), l2norm=True, scale=s["scale"],
            d_q=at, d_k=at + kw * size, d_v=at + 2 * kw * size, stride=qkv.shape[1],
            d_g=s["g"].data_ptr(), d_beta=s["beta"].data_ptr(),
            seq_start=None if max(s["lens"]) == 1 and min(s["lens"]) == 1 else _starts(s["lens"]),
            d_state_in=[s["state"][i].data_ptr() for i in range(n)],
            d_state_out=[s["new_state"][i].data_ptr() for i in range(n)], d_out=s["out"].data_ptr())
    ctx.gated_delta_dev(s["plan"])
    return {"out": s["out"], "state": s["new_state"]}


def _own_cache(ctx, s):
    c = s["case"]
    return ctx.kv_cache(d_k=s["k"].data_ptr(), d_v=s["v"].data_ptr(), d_k_scale=s["k_scale"].data_ptr(),
                        d_v_scale=s["v_scale"].data_ptr(), n_pages=s["n_pages"], page_tokens=c["page"],
                        kv_heads=c["kv_heads"], head_dim=c["head_dim"])


def _own_attn(s):
    ctx = _ctx()
    if "plan" not in s:
        c = s["case"]
        s["plan"] = ctx.attn_args(
            cache=_own_cache(ctx, s), n_seq=len(s["rows"]), q_heads=c["q_heads"], dtype=_code(c), scale=s["scale"],
            d_q=s["q"].data_ptr(), q_stride=c["q_heads"] * c["head_dim"],
            seq_start=None if max(s["rows"]) == 1 else _starts(s["rows"]), d_len=s["len"].data_ptr(),
            d_pages=s["pages"].data_ptr(), max_pages=s["pages"].shape[1], max_len=max(s["ctx"]),
            d_out=s["out"].data_ptr())
    ctx.attn_dev(s["plan"])
    return s["out"]


def _own_append(s):
    ctx = _ctx()
    if "plan" not in s:
        c = s["case"]
        cache, width = _own_cache(ctx, s), c["kv_heads"] * c["head_dim"]
        more = dict(cache=cache, n_seq=len(s["rows"]), k_stride=width, v_stride=width, d_len=s["len"].data_ptr(),
                    d_pages=s["pages"].data_ptr(), max_pages=s["pages"].shape[1])
        s["plan"] = ctx.kv_args(dtype=_code(c), d_k=s["new_k"].data_ptr(), d_v=s["new_v"].data_ptr(),
                                seq_start=_starts(s["rows"]), **more)
        s["read"] = ctx.kv_args(dtype=0, d_k=s["k_out"].data_ptr(), d_v=s["v_out"].data_ptr(),
                                seq_start=_starts(s["back"]), **more)
    ctx.kv_append_dev(s["plan"])
    ctx.kv_read_dev(s["read"])
    return {"k": s["k_out"], "v": s["v_out"]}


def _own_logprobs(s):
    n = s["case"]["top"]
    _ctx().logprobs_dev(s["logits"].data_ptr(), s["logits"].shape[0], s["logits"].shape[1], s["logits"].shape[1],
                        s["tokens"].data_ptr(), n, s["logprob"].data_ptr(), s["entropy"].data_ptr(),
                        s["ids"].data_ptr() if n else None, s["top"].data_ptr() if n else None)
    return {"logprob": s["logprob"], "entropy": s["entropy"], "ids": s["ids"], "top": s["top"]}


# ----------------------------------------------------------------------------------- plain forms
def _rows_of(counts, device="cuda"):
    """(sequence, place in it) of every row of a ragged batch."""
    c = torch.tensor(counts, device=device)
    seq = torch.repeat_interleave(torch.arange(len(counts), device=device), c, output_size=sum(counts))
    first = torch.tensor(_starts(counts)[:-1], device=device)
    return seq, torch.arange(sum(counts), device=device) - first[seq]


def _gdn_operands(s, dtype):
    """q, k, v [tokens][value heads][...], normalised, in `dtype`."""
    c = s["case"]
    hk, hv, dk, dv = c["k_heads"], c["v_heads"], c["k_dim"], c["v_dim"]
    x = s["qkv"].to(dtype)
    q, k, v = x[:, :hk * dk].view(-1, hk, dk), x[:, hk * dk:2 * hk * dk].view(-1, hk, dk), x[:, 2 * hk * dk:].view(-1, hv, dv)
    q = q * torch.rsqrt((q * q).sum(-1, keepdim=True) + 1e-6) * s["scale"]
    k = k * torch.rsqrt((k * k).sum(-1, keepdim=True) + 1e-6)
    of = torch.arange(hv, device=x.device) // (hv // hk)
    return q[:, of], k[:, of], v


def _plain_gdn(s):
    q, k, v = _gdn_operands(s, torch.float32)
    lens = s["lens"]
    if max(lens) == 1 and min(lens) == 1:
        st = s["state"] * torch.exp(s["g"])[..., None, None]
        u = (v - (st * k[:, :, None, :]).sum(-1)) * s["beta"][..., None]
        st = st + u[..., :, None] * k[..., None, :]
        return {"out": (st * q[:, :, None, :]).sum(-1).to(s["out"].dtype), "state": st}
    # chunks of 64 tokens, sequences padded with tokens that change nothing (no decay, beta 0)
    C, n, hv = 64, len(lens), v.shape[1]
    seq, at = _rows_of(lens)
    nc = -(-max(lens) // C)

    def pad(x):
        full = torch.zeros(n, nc * C, *x.shape[1:], device=x.device)
        full[seq, at] = x
        return full.view(n, nc, C, *x.shape[1:]).transpose(2, 3)   # [seq][chunk][head][token]...

    q, k, v, b = pad(q), pad(k), pad(v), pad(s["beta"][..., None])
    cum = pad(s["g"][..., None]).double().cumsum(3)                # decay since the chunk's start
    ratio = cum - cum.transpose(3, 4)                              # log decay from token j to token i
    low = torch.ones(C, C, dtype=torch.bool, device="cuda").tril()
    ratio = torch.exp(torch.where(low, ratio, torch.zeros_like(ratio)).float()) * low
    strict = low.tril(-1)
    a = b * (k @ k.transpose(3, 4).contiguous()) * ratio * strict
    t = torch.eye(C, device="cuda").expand(n, nc, hv, C, C).clone()
    for i in range(1, C):   # (1 + a)^-1, row by row
        t[..., i, :i] = -(a[..., i:i + 1, :i] @ t[..., :i, :i])[..., 0, :]
    e = torch.exp(cum.float())
    w, u = t @ (b * e * k), t @ (b * v)
    inside = (q @ k.transpose(3, 4).contiguous()) * ratio
    qe = q * e
    ke = (k * torch.exp((cum[..., -1:, :] - cum).float())).transpose(3, 4).contiguous()
    end = torch.exp(cum[..., -1, 0].float())
    st = s["state"].transpose(2, 3).contiguous()                   # [seq][head][k_dim][v_dim]
    out = []
    for i in range(nc):
        fresh = u[:, i] - w[:, i] @ st
        out.append(qe[:, i] @ st + inside[:, i] @ fresh)
        st = st * end[:, i, :, None, None] + ke[:, i] @ fresh
    out = torch.stack(out, 1).transpose(2, 3).reshape(n, nc * C, hv, -1)[seq, at]
    return {"out": out.to(s["out"].dtype), "state": st.transpose(2, 3).contiguous()}


def _cached(s, dtype):
    """Keys and values [seq][kv head][token][dim] of every table entry, as the codes stand for them."""
    c = s["case"]
    p = s["pages"].clamp(min=0).long()
    k = s["k"][p].to(dtype) * s["k_scale"][p].to(dtype)[..., None, None]      # [seq][page][head][token][dim]
    v = s["v"][p].to(dtype) * s["v_scale"][p].to(dtype)[..., None, None]      # [seq][page][head][dim][token]
    n, kv, d = p.shape[0], c["kv_heads"], c["head_dim"]
    return (k.permute(0, 2, 1, 3, 4).reshape(n, kv, -1, d), v.permute(0, 2, 1, 4, 3).reshape(n, kv, -1, d))


def _plain_attn(s):
    c = s["case"]
    k, v = _cached(s, torch.float32)
    n, kv, length, d = k.shape
    group = c["q_heads"] // kv
    seq, at = _rows_of(s["rows"])
    most = max(s["rows"])
    q = torch.zeros(n, most, c["q_heads"], d, device="cuda")
    q[seq, at] = s["q"].float()
    q = q.view(n, most, kv, group, d).permute(0, 2, 3, 1, 4).reshape(n, kv, group * most, d)
    score = (q @ k.transpose(2, 3).contiguous()) * s["scale"]
    rows = torch.tensor(s["rows"], device="cuda")
    last = (s["len"].long() - rows)[:, None] + torch.arange(most, device="cuda")      # a row's last key
    see = torch.arange(length, device="cuda")[None, None, :] <= last[..., None]
    score = score.view(n, kv, group, most, length).masked_fill(~see[:, None, None], float("-inf"))
    e = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-3e38))
    total = e.sum(-1, keepdim=True)
    o = (e.view(n, kv, group * most, length) @ v).view(n, kv, group, most, d) / total
    return o.permute(0, 3, 1, 2, 4).reshape(n, most, c["q_heads"], d)[seq, at].to(s["out"].dtype)


def _plain_append(s):
    c = s["case"]
    P, rows, ctx = c["page"], s["rows"], s["ctx"]
    seq, at = _rows_of(rows)
    start = s["len"].long() - torch.tensor(rows, device="cuda")
    pos = start[seq] + at
    slot = s["pages"][seq, pos // P].long()                                  # page of every new row
    old = torch.zeros(s["n_pages"], dtype=torch.long, device="cuda")          # tokens a page keeps
    head = s["pages"][torch.arange(len(rows), device="cuda"), start.clamp(min=0) // P].long()
    old[head] = start % P
    touched = torch.zeros(s["n_pages"], dtype=torch.bool, device="cuda")
    touched[slot] = True
    kept = torch.arange(P, device="cuda")[None, :] < old[:, None]             # [page][token]

    def write(codes, scales, x, token_axis):
        x = x.float()
        amax = torch.zeros(s["n_pages"], c["kv_heads"], device="cuda")
        amax = amax.scatter_reduce(0, slot[:, None].expand(-1, c["kv_heads"]), x.abs().amax(-1), "amax")
        before = torch.where((old > 0)[:, None], scales, torch.zeros_like(scales))
        after = torch.where(touched[:, None], torch.maximum(before, amax / 127.0), scales)
        div = torch.where(after > 0, after, torch.ones_like(after)).double()[..., None, None]
        again = torch.round(codes.double() * scales.double()[..., None, None] / div).to(torch.int8)
        keep = kept[:, None, :, None] if token_axis == 2 else kept[:, None, None, :]
        codes.copy_(torch.where(keep & touched[:, None, None, None], again, codes))
        new = torch.round(x.double() / div[slot][..., 0]).clamp(-127, 127).to(torch.int8)
        if token_axis == 2:
            codes[slot, :, pos % P] = new
        else:
            codes[slot, :, :, pos % P] = new
        scales.copy_(after)

    write(s["k"], s["k_scale"], s["new_k"], 2)
    write(s["v"], s["v_scale"], s["new_v"], 3)
    seq, at = _rows_of(s["back"])
    pos = s["len"].long()[seq] - torch.tensor(s["back"], device="cuda")[seq] + at
    slot = s["pages"][seq, pos // P].long()
    return {"k": s["k"][slot, :, pos % P].float() * s["k_scale"][slot][..., None],
            "v": s["v"][slot, :, :, pos % P].float() * s["v_scale"][slot][..., None]}


def _plain_logprobs(s):
    x, n = s["logits"], s["case"]["top"]
    top, first = x.max(-1, keepdim=True)
    d = x - top
    e = torch.exp(d)
    rest = e.scatter(1, first, 0.0).sum(-1)                   # all but the maximum's own 1
    log_z = torch.log1p(rest)
    given = d.gather(1, s["tokens"].long()[:, None])[:, 0] - log_z
    entropy = log_z - (e * d).sum(-1) / (1.0 + rest)
    # a stable sort keeps equal values in the order of their indices
    if n:
        val, ids = torch.sort(x, dim=-1, descending=True, stable=True)
        val, ids = val[:, :n], ids[:, :n]
    else:
        val, ids = x[:, :0], torch.empty(x.shape[0], 0, dtype=torch.int64, device="cuda")
    return {"logprob": given, "entropy": entropy, "ids": ids.to(torch.int32),
            "top": val - top - log_z[:, None]}


# ------------------------------------------------------------------------------ work and definition
def work(case):
    size = 2 if case.get("dtype") == BF16 else 4
    if case["op"] == "gdn":
        lens = _ints(case["lens"])
        hv, cell = case["v_heads"], case["k_dim"] * case["v_dim"]
        row = (2 * case["k_heads"] * case["k_dim"] + 2 * hv * case["v_dim"]) * size + 8 * hv
        return {"bytes": sum(lens) * row + 8 * len(lens) * hv * cell, "flops": 8 * sum(lens) * hv * cell}
    if case["op"] == "logprobs":
        return {"bytes": case["rows"] * (4 * case["vocab"] + 12 + 8 * case["top"]), "flops": 6 * case["rows"] * case["vocab"]}
    rows, ctx, kv, d = _ints(case["rows"]), _ints(case["ctx"]), case["kv_heads"], case["head_dim"]
    if case["op"] == "append":
        back = sum(r + (c - r) % case["page"] for r, c in zip(rows, ctx))
        return {"bytes": kv * d * (2 * size * sum(rows) + 2 * sum(rows) + 10 * back), "flops": 4 * kv * d * sum(rows)}
    pairs = sum(r * (c - r) + r * (r + 1) // 2 for r, c in zip(rows, ctx))
    return {"bytes": sum(ctx) * kv * (2 * d + 8 / case["page"]) + 2 * sum(rows) * case["q_heads"] * d * size,
            "flops": 4 * pairs * case["q_heads"] * d}


def exact(case, seed):
    s = prepare(case, seed)
    return {"gdn": _exact_gdn, "attn": _exact_attn, "append": _exact_append, "logprobs": _exact_logprobs}[case["op"]](s)


def _exact_gdn(s):
    """The recurrence token by token in 64 bits."""
    c, lens = s["case"], s["lens"]
    rep = c["v_heads"] // c["k_heads"]
    x = s["qkv"].double()
    kw = c["k_heads"] * c["k_dim"]

    def unit(y):
        y = y.reshape(y.shape[0], c["k_heads"], c["k_dim"])
        return (y / (y.square().sum(-1, keepdim=True) + 1e-6).sqrt()).repeat_interleave(rep, 1)

    q, k, v = unit(x[:, :kw]), unit(x[:, kw:2 * kw]), x[:, 2 * kw:].reshape(-1, c["v_heads"], c["v_dim"])
    a, b = s["g"].double().exp(), s["beta"].double()
    out = torch.empty(v.shape, dtype=torch.float64, device="cuda")
    start = _starts(lens)
    state = s["state"].double()
    for t in range(max(lens)):
        live = [i for i, n in enumerate(lens) if n > t]
        idx = [start[i] + t for i in live]
        whole = len(live) == len(lens)
        st = state if whole else state[live]
        at = slice(idx[0], idx[0] + 1) if len(idx) == 1 else idx
        st = st * a[at][..., None, None]
        u = b[at][..., None] * (v[at] - torch.einsum("nhvk,nhk->nhv", st, k[at]))
        st = st + torch.einsum("nhv,nhk->nhvk", u, k[at])
        out[at] = torch.einsum("nhvk,nhk->nhv", st, q[at]) * s["scale"]
        if whole:
            state = st
        else:
            state[live] = st
    return {"out": out, "state": state}


def _exact_attn(s):
    """Softmax over each row's keys in 64 bits, one sequence and cache head at a time."""
    c, P = s["case"], s["case"]["page"]
    group = c["q_heads"] // c["kv_heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    start = _starts(s["rows"])
    for i, (r, n) in enumerate(zip(s["rows"], s["ctx"])):
        p = s["pages"][i, :-(-n // P)].long()
        for h in range(c["kv_heads"]):
            k = (s["k"][p, h].double() * s["k_scale"][p, h].double()[:, None, None]).reshape(-1, c["head_dim"])[:n]
            v = (s["v"][p, h].double() * s["v_scale"][p, h].double()[:, None, None]).transpose(1, 2).reshape(-1, c["head_dim"])[:n]
            hidden = torch.arange(n, device="cuda")[None, :] > (n - r) + torch.arange(r, device="cuda")[:, None]
            for j in range(h * group, (h + 1) * group):
                q = s["q"][start[i]:start[i + 1], j].double()
                z = torch.where(hidden, -math.inf, torch.mm(q, k.t()) * s["scale"])
                out[start[i]:start[i + 1], j] = torch.mm(torch.softmax(z, -1), v)
    return out


def _exact_append(s):
    """What the cache stands for afterwards, page by page, rounding decided in 64 bits."""
    c, P = s["case"], s["case"]["page"]
    found = {}
    for name, new, scales in (("k", s["new_k"], s["k_scale"]), ("v", s["new_v"], s["v_scale"])):
        got, row = [], 0
        for i, (r, n) in enumerate(zip(s["rows"], s["ctx"])):
            x = new[row:row + r].double()
            row += r
            pos = n - r
            while pos < n:
                page = int(s["pages"][i, pos // P])
                keep, take = pos % P, min(P - pos % P, n - pos)
                part, x = x[:take], x[take:]
                scale = (part.abs().amax((0, 2)) / 127.0).float()
                old = s[name][page] if name == "k" else s[name][page].transpose(1, 2)     # [head][token][dim]
                old = old[:, :keep].transpose(0, 1).double()
                if keep:
                    was = scales[page]
                    scale = torch.maximum(scale, was)
                    old = torch.round(old * was.double()[:, None] / scale.double()[:, None])
                codes = torch.cat([old, torch.round(part / scale.double()[:, None]).clamp(-127, 127)])
                got.append(codes * scale.double()[:, None])
                pos += take
        found[name] = torch.cat(got)
    return found


def _exact_logprobs(s):
    x = s["logits"].double()
    lp = torch.log_softmax(x, -1)
    n = s["case"]["top"]
    top = torch.empty(x.shape[0], n, dtype=torch.float64, device="cuda")
    if n:
        top = lp.topk(n, -1, sorted=True).values
    return {"logprob": lp.gather(1, s["tokens"].long()[:, None])[:, 0], "entropy": -(lp.exp() * lp).sum(-1), "ids": None,
            "top": top}
