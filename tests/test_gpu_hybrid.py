"""The token mixers and the log probabilities between the framework's own products, as a hybrid
model's forward pass uses them: embedding lookup, a gated-delta layer (4-bit projections around
fm_gated_delta_dev), an attention layer over the 8-bit cache (projections, append, attention), the
vocabulary projection and the log probabilities — a prompt first, then single tokens, all on the
context's stream.  Each stage is checked in 64 bits on what the stage before it left."""
import numpy as np
import pytest

from finchmoe_amd import binding as fb
from finchmoe_amd import formats as F
from . import mix_ref as R
from .conftest import assert_parity

pytestmark = pytest.mark.gpu

H, VOCAB = 256, 1000
HK, HV, DK, DV = 2, 4, 64, 64          # gated delta layer: q, k, v = 128 + 128 + 256
HQ, KV, D, PAGE = 8, 2, 64, 16         # attention layer


class Model:
    def __init__(self, hip, orc, seed):
        rng = np.random.default_rng(seed)
        self.hip, self.w, self.t = hip, {}, {}
        for name, rows, cols, bits in (("embed", VOCAB, H, 8), ("qkv", 2 * HK * DK + HV * DV, H, 4), ("out", H, HV * DV, 4),
                                       ("q", HQ * D, H, 4), ("kv", 2 * KV * D, H, 4), ("o", H, HQ * D, 4), ("head", VOCAB, H, 8)):
            W, S, B = F.synth_affine_tensor(rng, rows, cols, bits, "bf16")[:3]
            _, w32 = orc.dequant_affine(W, S, B, rows, cols, bits)
            self.w[name] = np.asarray(w32, np.float64).reshape(rows, cols)
            self.t[name] = hip.tensor_register(W, S, B, rows, cols, bits=bits)

    def mv(self, name, x, out):
        self.hip.matvec_prefill_dev(self.t[name], x.data_ptr(), out.data_ptr(), x.shape[0])
        return out

    def close(self):
        for t in self.t.values():
            self.hip.tensor_release(t)


def test_prompt_then_tokens(hip, orc):
    import torch
    m = Model(hip, orc, 71)
    stream = torch.cuda.ExternalStream(hip.stream())
    rng = torch.Generator().manual_seed(72)
    prompt, steps, max_pages = 83, 5, 7
    total = prompt + steps
    with torch.cuda.stream(stream):
        tokens = torch.randint(0, VOCAB, (total,), generator=rng).to(torch.int32).cuda()
        gate = -torch.nn.functional.softplus(torch.randn(total, HV, generator=rng) - 2).cuda()
        beta = torch.sigmoid(torch.randn(total, HV, generator=rng)).cuda()
        state = torch.zeros(HV, DV, DK, device="cuda")
        pool = (torch.zeros(8, KV, PAGE, D, dtype=torch.int8, device="cuda"), torch.zeros(8, KV, D, PAGE, dtype=torch.int8, device="cuda"),
                torch.zeros(8, KV, device="cuda"), torch.zeros(8, KV, device="cuda"))
        table = torch.tensor([[4, 1, 7, 0, 3, 6, 2]], dtype=torch.int32, device="cuda")
        length = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache = hip.kv_cache(d_k=pool[0].data_ptr(), d_v=pool[1].data_ptr(), d_k_scale=pool[2].data_ptr(), d_v_scale=pool[3].data_ptr(),
                         n_pages=8, page_tokens=PAGE, kv_heads=KV, head_dim=D)
    ref_state = torch.zeros(1, HV, DV, DK, dtype=torch.float64)
    ref_pool = tuple(t.cpu() for t in pool)
    at = 0
    for n in [prompt] + [1] * steps:
        def new(*shape, dtype=torch.float32):
            return torch.empty(*shape, dtype=dtype, device="cuda")
        with torch.cuda.stream(stream):
            ids = tokens[at:at + n]
            x = new(n, H)
            hip.embed_lookup_dev(m.t["embed"], ids.data_ptr(), n, x.data_ptr())
            qkv = torch.nn.functional.silu(m.mv("qkv", x, new(n, 2 * HK * DK + HV * DV)))
            mixed = new(n, HV, DV)
            hip.gated_delta_dev(hip.gated_delta_args(
                n_seq=1, k_heads=HK, v_heads=HV, k_dim=DK, v_dim=DV, l2norm=True, scale=DK ** -0.5, stride=qkv.shape[1],
                d_q=qkv.data_ptr(), d_k=qkv.data_ptr() + 4 * HK * DK, d_v=qkv.data_ptr() + 8 * HK * DK,
                d_g=gate[at:].data_ptr(), d_beta=beta[at:].data_ptr(), seq_start=[0, n],
                d_state_in=[state.data_ptr()], d_state_out=[state.data_ptr()], d_out=mixed.data_ptr()))
            x1 = x + m.mv("out", mixed.view(n, -1), new(n, H))
            q, kv = m.mv("q", x1, new(n, HQ * D)), m.mv("kv", x1, new(n, 2 * KV * D))
            length += n
            rows = dict(cache=cache, n_seq=1, d_len=length.data_ptr(), d_pages=table.data_ptr(), max_pages=max_pages)
            hip.kv_append_dev(hip.kv_args(d_k=kv.data_ptr(), d_v=kv.data_ptr() + 4 * KV * D, k_stride=2 * KV * D,
                                          v_stride=2 * KV * D, seq_start=[0, n], **rows))
            seen = new(n, HQ, D)
            hip.attn_dev(hip.attn_args(q_heads=HQ, d_q=q.data_ptr(), max_len=total, d_out=seen.data_ptr(), scale=D ** -0.5,
                                       seq_start=[0, n], **rows))
            x2 = x1 + m.mv("o", seen.view(n, -1), new(n, H))
            logits = m.mv("head", x2, new(n, VOCAB))
            lp, entropy, top, top_lp = new(n), new(n), new(n, 4, dtype=torch.int32), new(n, 4)
            follow = tokens[at + 1:at + n + 1] if at + n < total else torch.zeros(n, dtype=torch.int32, device="cuda")
            follow = torch.nn.functional.pad(follow, (0, n - follow.numel())).contiguous()
            hip.logprobs_dev(logits.data_ptr(), n, VOCAB, VOCAB, follow.data_ptr(), 4, lp.data_ptr(), entropy.data_ptr(),
                             top.data_ptr(), top_lp.data_ptr())
        hip.sync()

        def num(t):
            return t.detach().cpu().double().numpy()
        what = "tokens %d.." % at
        assert_parity(num(x), m.w["embed"][ids.cpu().numpy()], what + " embedding")
        pre = num(x) @ m.w["qkv"].T
        assert_parity(num(qkv), pre / (1 + np.exp(-pre)), what + " projection")
        c = qkv.cpu()
        ref, ref_state = R.gated_delta(c[:, :128].reshape(n, HK, DK), c[:, 128:256].reshape(n, HK, DK), c[:, 256:].reshape(n, HV, DV),
                                       gate[at:at + n].cpu(), beta[at:at + n].cpu(), ref_state, [n], DK ** -0.5, True)
        tol = R.U24 * (DK + 16) * (at + n) ** 0.5
        R.close(mixed, ref, tol * float(ref.abs().max()), 0.0, what + " mixer")
        R.close(state[None], ref_state, tol * float(ref_state.abs().max()), 0.0, what + " state")
        assert_parity(num(x1), num(x) + num(mixed).reshape(n, -1) @ m.w["out"].T, what + " layer 1")
        assert_parity(num(kv), num(x1) @ m.w["kv"].T, what + " keys and values")
        ck = kv.cpu().reshape(n, 2, KV, D)
        ref_pool = R.append(ref_pool + (PAGE,), table.cpu(), [at + n], [n], ck[:, 0], ck[:, 1])
        for got, want in zip(pool, ref_pool):
            assert torch.equal(got.cpu(), want), what
        ref, most, vmax = R.attention(q.cpu().reshape(n, HQ, D), ref_pool + (PAGE,), table.cpu(), [at + n], [n], D ** -0.5, total)
        R.close(seen, ref, vmax * R.U24 * (2 * most * (D + 8) + 8 + total / 32 + 40), 0.0, what + " attention")
        assert_parity(num(x2), num(x1) + num(seen).reshape(n, -1) @ m.w["o"].T, what + " layer 2")
        assert_parity(num(logits), num(x2) @ m.w["head"].T, what + " logits")
        r_lp, r_en, r_ids, r_top = R.logprobs(logits.cpu(), follow.cpu(), 4)
        R.close(lp, r_lp, 96 * R.U24, 2 * R.U24, what + " log probabilities")
        R.close(entropy, r_en, R.U24 * (128 + 4 * np.log(VOCAB) ** 2), 0.0, what + " entropy")
        assert torch.equal(top.cpu(), r_ids), what
        R.close(top_lp, r_top, 96 * R.U24, 2 * R.U24, what + " top")
        at += n
    m.close()


def _calls(hip, n, prompt):
    """One token mixer call of each kind over static buffers: (buffers that change, outputs, submit)."""
    import torch
    g = torch.Generator().manual_seed(n + prompt)
    rows = prompt if prompt else n
    starts = [0, prompt] if prompt else None
    seqs = 1 if prompt else n
    qkv = torch.randn(rows, 2 * HK * DK + HV * DV, generator=g).cuda()
    gate, beta = -torch.rand(rows, HV, generator=g).cuda(), torch.rand(rows, HV, generator=g).cuda()
    st_in, st_out = torch.randn(seqs, HV, DV, DK, generator=g).cuda(), torch.zeros(seqs, HV, DV, DK, device="cuda")
    mixed = torch.zeros(rows, HV, DV, device="cuda")
    a1 = hip.gated_delta_args(n_seq=seqs, k_heads=HK, v_heads=HV, k_dim=DK, v_dim=DV, l2norm=True, scale=0.1, stride=qkv.shape[1],
                              d_q=qkv.data_ptr(), d_k=qkv.data_ptr() + 4 * HK * DK, d_v=qkv.data_ptr() + 8 * HK * DK,
                              d_g=gate.data_ptr(), d_beta=beta.data_ptr(), seq_start=starts,
                              d_state_in=[s.data_ptr() for s in st_in], d_state_out=[s.data_ptr() for s in st_out],
                              d_out=mixed.data_ptr())
    pages = seqs * 20
    k8, v8 = torch.zeros(pages, KV, PAGE, D, dtype=torch.int8, device="cuda"), torch.zeros(pages, KV, D, PAGE, dtype=torch.int8, device="cuda")
    ks, vs = torch.zeros(pages, KV, device="cuda"), torch.zeros(pages, KV, device="cuda")
    table = torch.arange(pages, dtype=torch.int32, device="cuda").view(seqs, 20).contiguous()
    length = torch.full((seqs,), rows if prompt else 1, dtype=torch.int32, device="cuda")
    q, kv = torch.randn(rows, HQ * D, generator=g).cuda(), torch.randn(rows, 2 * KV * D, generator=g).cuda()
    seen = torch.zeros(rows, HQ, D, device="cuda")
    cache = hip.kv_cache(d_k=k8.data_ptr(), d_v=v8.data_ptr(), d_k_scale=ks.data_ptr(), d_v_scale=vs.data_ptr(), n_pages=pages,
                         page_tokens=PAGE, kv_heads=KV, head_dim=D)
    common = dict(cache=cache, n_seq=seqs, seq_start=starts, d_len=length.data_ptr(), d_pages=table.data_ptr(), max_pages=20)
    a2 = hip.kv_args(d_k=kv.data_ptr(), d_v=kv.data_ptr() + 4 * KV * D, k_stride=2 * KV * D, v_stride=2 * KV * D, **common)
    a3 = hip.attn_args(q_heads=HQ, d_q=q.data_ptr(), max_len=320, d_out=seen.data_ptr(), scale=0.2, **common)
    logits = torch.randn(rows, 5000, generator=g).cuda()
    tok = torch.zeros(rows, dtype=torch.int32, device="cuda")
    lp, ids, top = torch.zeros(rows, device="cuda"), torch.zeros(rows, 3, dtype=torch.int32, device="cuda"), torch.zeros(rows, 3, device="cuda")

    def submit():
        hip.gated_delta_dev(a1)
        hip.kv_append_dev(a2)
        hip.attn_dev(a3)
        hip.logprobs_dev(logits.data_ptr(), rows, 5000, 5000, tok.data_ptr(), 3, lp.data_ptr(), None, ids.data_ptr(), top.data_ptr())
    submit.keep = (gate, beta, st_in, table, tok)      # (the descriptors hold addresses only)
    need = max(hip.gated_delta_ws_bytes(a1), hip.attn_ws_bytes(a3), hip.logprobs_ws_bytes(rows, 5000, 3))
    return (qkv, q, kv, logits), (mixed, st_out, seen, lp, ids, top, k8, v8, ks, vs), length, submit, need


@pytest.mark.parametrize("n,prompt", [(3, 0), (1, 90)])
def test_replayed_from_a_graph(n, prompt):
    """captured once, replayed with new inputs and growing sequences between eager calls"""
    import ctypes as C
    import torch
    from finchmoe_amd import FinchHip
    from .test_gpu_graph import _hip
    lib = _hip()
    hip = FinchHip(0)
    try:
        change, outs, length, submit, need = _calls(hip, n, prompt)
        hip.reserve(workspace_bytes=need)
        torch.cuda.synchronize()
        stream, graph, gexec = C.c_void_p(hip.stream()), C.c_void_p(), C.c_void_p()
        assert lib.hipStreamBeginCapture(stream, 2) == 0
        submit()
        assert lib.hipStreamEndCapture(stream, C.byref(graph)) == 0
        assert lib.hipGraphInstantiate(C.byref(gexec), graph, None, None, 0) == 0
        rng = torch.Generator().manual_seed(5)
        for rep in range(5):
            for t in change:
                t.copy_(torch.randn(t.shape, generator=rng))
            before = [o.clone() for o in outs]
            torch.cuda.synchronize()
            submit()
            hip.sync()
            eager = [o.clone() for o in outs]
            for o, b in zip(outs, before):      # the cache and the states as they were
                o.copy_(b)
            torch.cuda.synchronize()
            assert lib.hipGraphLaunch(gexec, stream) == 0
            hip.sync()
            for i, (o, e) in enumerate(zip(outs, eager)):
                assert torch.equal(o, e), (rep, i)
            if not prompt:
                length += torch.tensor([7, 60, 1], dtype=torch.int32, device="cuda")
        lib.hipGraphExecDestroy(gexec)
        lib.hipGraphDestroy(graph)
    finally:
        hip.close()


def test_workspace_may_not_grow_under_a_graph():
    import ctypes as C
    import torch
    from finchmoe_amd import FinchError, FinchHip
    from .test_gpu_graph import _hip
    lib = _hip()
    hip = FinchHip(0)
    try:
        _, _, _, submit, need = _calls(hip, 1, 90)
        torch.cuda.synchronize()
        stream, graph = C.c_void_p(hip.stream()), C.c_void_p()
        assert lib.hipStreamBeginCapture(stream, 2) == 0
        with pytest.raises(FinchError) as e:
            submit()
        assert e.value.status == fb.ERR_STATE and "fm_reserve" in str(e.value)
        lib.hipStreamEndCapture(stream, C.byref(graph))
        lib.hipGraphDestroy(graph)
        hip.release_graphs()
        hip.reserve(workspace_bytes=need)
        submit()
        hip.sync()
    finally:
        hip.close()


def test_two_contexts_at_once():
    """two contexts' calls in flight together (own streams, own workspaces) give what each gives alone"""
    import torch
    from finchmoe_amd import FinchHip
    a, b = FinchHip(0), FinchHip(0)
    try:
        ca, cb = _calls(a, 1, 200), _calls(b, 1, 150)
        torch.cuda.synchronize()
        want = []
        for c, hip in ((ca, a), (cb, b)):
            c[3]()
            hip.sync()
            want.append([o.clone() for o in c[1]])
        torch.cuda.synchronize()
        for _ in range(5):
            ca[3]()
            cb[3]()
        a.sync()
        b.sync()
        for c, w in zip((ca, cb), want):
            for o, e in zip(c[1], w):
                assert torch.equal(o, e)
    finally:
        a.close()
        b.close()
