"""fm_gated_delta_dev against the recurrence in 64 bits.

Tolerance of fp32 outputs, relative to the tensor's largest value: a token's sums over k_dim are off by at
most (k_dim + 16) half steps of the magnitudes they add (products, normalisation, decay and update
are the 16), tokens' roundings are independent of each other and a step does not enlarge what is
there (decay <= 1, |1 - beta k k^T| <= 1 for unit k), so T tokens add sqrt(T) of that.  bf16 outputs
add half a step of bf16."""
import numpy as np
import pytest

from finchmoe_amd import binding as fb
from . import mix_ref as R

pytestmark = pytest.mark.gpu


def _inputs(seed, lens, hk, hv, dk, dv, dtype, pad=0, decay=-3.0):
    import torch
    g = torch.Generator().manual_seed(seed)
    n = sum(lens)
    width = 2 * hk * dk + hv * dv + pad
    rows = torch.nn.functional.silu(torch.randn(n, width, generator=g)).to(dtype)
    a = torch.log(1 + 15 * torch.rand(hv, generator=g))
    gate = -a.exp() * torch.nn.functional.softplus(torch.randn(n, hv, generator=g) + decay)
    beta = torch.sigmoid(torch.randn(n, hv, generator=g))
    state = 0.3 * torch.randn(len(lens), hv, dv, dk, generator=g)
    return rows, gate, beta, state


def _split(rows, hk, hv, dk, dv):
    n, kw = rows.shape[0], hk * dk
    return (rows[:, :kw].reshape(n, hk, dk), rows[:, kw:2 * kw].reshape(n, hk, dk),
            rows[:, 2 * kw:2 * kw + hv * dv].reshape(n, hv, dv))


def _call(hip, rows, gate, beta, state, lens, hk, hv, dk, dv, l2norm, scale, in_place=False, no_state=False, one_row=False,
          calls=1):
    import torch
    bf = rows.dtype == torch.bfloat16
    d = rows.cuda()
    size, kw = d.element_size(), hk * dk
    dg, db, ds = gate.cuda(), beta.cuda(), state.cuda()
    new = ds if in_place else torch.full_like(ds, float("nan"))
    out = torch.full((max(1, rows.shape[0]), hv, dv), float("nan"), dtype=rows.dtype, device="cuda")
    n = len(lens)
    a = hip.gated_delta_args(
        n_seq=n, k_heads=hk, v_heads=hv, k_dim=dk, v_dim=dv, dtype=fb.DTYPE_BF16 if bf else fb.DTYPE_F32,
        l2norm=l2norm, scale=scale, d_q=d.data_ptr(), d_k=d.data_ptr() + kw * size, d_v=d.data_ptr() + 2 * kw * size,
        stride=d.shape[1], d_g=dg.data_ptr(), d_beta=db.data_ptr(), seq_start=None if one_row else R.starts(lens),
        d_state_in=None if no_state else [ds[i].data_ptr() for i in range(n)],
        d_state_out=[new[i].data_ptr() for i in range(n)], d_out=out.data_ptr())
    torch.cuda.synchronize()
    for _ in range(calls):
        hip.gated_delta_dev(a)
    hip.sync()
    return out[:rows.shape[0]].float().cpu(), new.cpu()


def _check(got, new, ref, ref_s, lens, dk, bf, what):
    T = max(max(lens), 1)
    tol = R.U24 * (dk + 16) * T ** 0.5
    R.close(got, ref, tol * float(ref.abs().max()) if ref.numel() else 0.0, R.U_BF16 if bf else 0.0, what + " out")
    R.close(new, ref_s, tol * float(ref_s.abs().max()), 0.0, what + " state")


SHAPES = [(1, 1, 64, 16), (2, 4, 128, 128), (1, 3, 64, 80), (2, 2, 128, 256), (4, 4, 128, 48)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("hk,hv,dk,dv", SHAPES)
@pytest.mark.parametrize("lens", [[1], [1, 1, 1], [2], [5, 0, 1], [23], [24], [63], [64], [65], [130, 17], [200]])
def test_against_the_recurrence(hip, lens, hk, hv, dk, dv, dtype):
    import torch
    dt = getattr(torch, dtype)
    rows, gate, beta, state = _inputs(len(lens) * 100 + sum(lens), lens, hk, hv, dk, dv, dt)
    q, k, v = _split(rows, hk, hv, dk, dv)
    scale = dk ** -0.5
    ref, ref_s = R.gated_delta(q, k, v, gate, beta, state, lens, scale, True)
    got, new = _call(hip, rows, gate, beta, state, lens, hk, hv, dk, dv, True, scale)
    _check(got, new, ref, ref_s, lens, dk, dt == torch.bfloat16, "lens %s" % lens)


@pytest.mark.parametrize("lens", [[1] * 7, [33, 100]])
def test_without_normalisation_and_other_scale(hip, lens):
    """keys of unit length already; queries of any length"""
    import torch
    hk, hv, dk, dv = 2, 4, 128, 64
    rows, gate, beta, state = _inputs(7, lens, hk, hv, dk, dv, torch.float32)
    q, k, v = _split(rows, hk, hv, dk, dv)
    k /= k.square().sum(-1, keepdim=True).sqrt()        # (a view: writes the rows)
    ref, ref_s = R.gated_delta(q, k, v, gate, beta, state, lens, 0.7, False)
    got, new = _call(hip, rows, gate, beta, state, lens, hk, hv, dk, dv, False, 0.7)
    _check(got, new, ref, ref_s, lens, dk, False, "no norm")


@pytest.mark.parametrize("lens", [[1], [1, 1], [90]])
def test_in_place_without_state_and_padded_rows(hip, lens):
    import torch
    hk, hv, dk, dv = 2, 2, 64, 32
    rows, gate, beta, state = _inputs(8, lens, hk, hv, dk, dv, torch.float32, pad=12)
    q, k, v = _split(rows, hk, hv, dk, dv)
    ref, ref_s = R.gated_delta(q, k, v, gate, beta, state, lens, 1.0, True)
    got, new = _call(hip, rows, gate, beta, state, lens, hk, hv, dk, dv, True, 1.0, in_place=True)
    _check(got, new, ref, ref_s, lens, dk, False, "in place")
    ref, ref_s = R.gated_delta(q, k, v, gate, beta, torch.zeros_like(state), lens, 1.0, True)
    got, new = _call(hip, rows, gate, beta, state, lens, hk, hv, dk, dv, True, 1.0, no_state=True)
    _check(got, new, ref, ref_s, lens, dk, False, "no state")


def test_one_row_form_equals_starts(hip):
    import torch
    hk, hv, dk, dv, lens = 2, 4, 128, 128, [1] * 5
    rows, gate, beta, state = _inputs(9, lens, hk, hv, dk, dv, torch.bfloat16)
    a = _call(hip, rows, gate, beta, state, lens, hk, hv, dk, dv, True, 0.1, one_row=True)
    b = _call(hip, rows, gate, beta, state, lens, hk, hv, dk, dv, True, 0.1)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_calls_repeat_bit_for_bit(hip):
    import torch
    hk, hv, dk, dv, lens = 2, 4, 128, 128, [150, 3, 70]
    rows, gate, beta, state = _inputs(10, lens, hk, hv, dk, dv, torch.float32)
    a = _call(hip, rows, gate, beta, state, lens, hk, hv, dk, dv, True, 0.1)
    b = _call(hip, rows, gate, beta, state, lens, hk, hv, dk, dv, True, 0.1, calls=3)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("lens", [[3], [100], [129]])
def test_decay_of_any_size(hip, lens):
    """-inf and huge negative logarithms wipe the state, 0 keeps it; a strong decay early in a chunk must
    not cost later tokens their digits."""
    import torch
    hk, hv, dk, dv = 1, 4, 64, 64
    rows, gate, beta, state = _inputs(11, lens, hk, hv, dk, dv, torch.float32)
    n = sum(lens)
    gate[:, 0] = 0.0
    gate[n // 2, 1] = -float("inf")
    gate[:, 2] = -60.0
    gate[: n // 2, 3] = -95.0
    gate[n // 2:, 3] = -0.01
    q, k, v = _split(rows, hk, hv, dk, dv)
    ref, ref_s = R.gated_delta(q, k, v, gate, beta, state, lens, 1.0, True)
    got, new = _call(hip, rows, gate, beta, state, lens, hk, hv, dk, dv, True, 1.0)
    _check(got, new, ref, ref_s, lens, dk, False, "decay")
    for h in range(hv):   # each head by its own largest value
        tol = R.U24 * (dk + 16) * max(lens) ** 0.5
        R.close(got[:, h], ref[:, h], tol * float(ref[:, h].abs().max()), 0.0, "head %d" % h)


def test_correlated_keys_and_full_beta(hip):
    """the chunk's triangular system at its worst conditioned: one key direction, beta 1, no decay"""
    import torch
    hk, hv, dk, dv, lens = 1, 2, 128, 64, [192]
    rows, gate, beta, state = _inputs(12, lens, hk, hv, dk, dv, torch.float32)
    q, k, v = _split(rows, hk, hv, dk, dv)
    k.copy_(k[:1] + 0.05 * k)
    gate.zero_()
    beta.fill_(1.0)
    ref, ref_s = R.gated_delta(q, k, v, gate, beta, state, lens, 1.0, True)
    got, new = _call(hip, rows, gate, beta, state, lens, hk, hv, dk, dv, True, 1.0)
    _check(got, new, ref, ref_s, lens, dk, False, "correlated")


def test_nan_stays_in_its_head_and_sequence(hip):
    import torch
    hk, hv, dk, dv, lens = 2, 2, 64, 16, [70, 70]
    rows, gate, beta, state = _inputs(13, lens, hk, hv, dk, dv, torch.float32)
    gate[5, 1] = float("nan")
    got, new = _call(hip, rows, gate, beta, state, lens, hk, hv, dk, dv, True, 1.0)
    assert bool(torch.isfinite(got[:, 0]).all()) and bool(torch.isfinite(got[70:]).all())
    assert bool(torch.isnan(got[5:70, 1]).all()) and bool(torch.isnan(new[0, 1]).all())
    assert bool(torch.isfinite(new[1]).all()) and bool(torch.isfinite(new[0, 0]).all())


def test_many_sequences_in_several_launches(hip):
    import torch
    hk, hv, dk, dv = 1, 1, 64, 16
    lens = [1 + i % 3 for i in range(256)]
    rows, gate, beta, state = _inputs(14, lens, hk, hv, dk, dv, torch.float32)
    q, k, v = _split(rows, hk, hv, dk, dv)
    ref, ref_s = R.gated_delta(q, k, v, gate, beta, state, lens, 1.0, True)
    got, new = _call(hip, rows, gate, beta, state, lens, hk, hv, dk, dv, True, 1.0)
    _check(got, new, ref, ref_s, lens, dk, False, "256 sequences")


def test_windows_of_chunks(hip):
    """more chunks than one launch's workspace holds: 40 sequences of 32 heads, up to five chunks each"""
    import torch
    hk, hv, dk, dv = 16, 32, 128, 16
    lens = [100 + 5 * i for i in range(38)] + [7, 64]
    rows, gate, beta, state = _inputs(16, lens, hk, hv, dk, dv, torch.float32)
    q, k, v = _split(rows, hk, hv, dk, dv)
    ref, ref_s = R.gated_delta(q, k, v, gate, beta, state, lens, 1.0, True)
    got, new = _call(hip, rows, gate, beta, state, lens, hk, hv, dk, dv, True, 1.0)
    _check(got, new, ref, ref_s, lens, dk, False, "windows")
    got, new = _call(hip, rows, gate, beta, state, lens, hk, hv, dk, dv, True, 1.0, in_place=True)
    _check(got, new, ref, ref_s, lens, dk, False, "windows, in place")


def test_step_after_step_equals_the_prompt(hip):
    """A prompt in one call, and token by token with the state carried over: equal to rounding."""
    import torch
    hk, hv, dk, dv, T = 2, 4, 128, 128, 70
    rows, gate, beta, state = _inputs(15, [T], hk, hv, dk, dv, torch.float32)
    whole, end = _call(hip, rows, gate, beta, state, [T], hk, hv, dk, dv, True, 1.0)
    st, outs = state, []
    for t in range(T):
        o, st = _call(hip, rows[t:t + 1], gate[t:t + 1], beta[t:t + 1], st, [1], hk, hv, dk, dv, True, 1.0, one_row=True)
        outs.append(o)
    tol = 2 * R.U24 * (dk + 16) * T ** 0.5
    R.close(torch.cat(outs), whole, tol * float(whole.abs().max()), 0.0, "out")
    R.close(st, end, tol * float(end.abs().max()), 0.0, "state")


def test_refusals(hip):
    import torch
    z = torch.zeros(1 << 16, device="cuda")
    p = z.data_ptr()
    good = dict(n_seq=1, k_heads=1, v_heads=1, k_dim=64, v_dim=16, d_q=p, d_k=p, d_v=p, d_g=p, d_beta=p,
                d_state_out=[p + 65536], d_out=p + 131072)

    def status(**kw):
        with pytest.raises(fb.FinchError) as e:
            hip.gated_delta_dev(hip.gated_delta_args(**dict(good, **kw)))
        return e.value.status

    assert status(k_dim=96) == fb.ERR_UNSUPPORTED and status(v_dim=24) == fb.ERR_UNSUPPORTED
    assert status(v_heads=3, k_heads=2) == fb.ERR_ARG and status(d_q=p + 4) == fb.ERR_ARG
    assert status(d_state_out=[0]) == fb.ERR_ARG and status(stride=62) == fb.ERR_ARG
    assert status(n_seq=2, d_state_out=[p + 65536] * 2) == fb.ERR_ARG
    assert status(d_state_in=[p + 65536 + 16]) == fb.ERR_ARG
    hip.gated_delta_dev(hip.gated_delta_args(**good))
    hip.sync()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("lens", [[9000] + [64] * 7 + [3], [64] * 6 + [9000, 7] + [24] * 30, [100] * 140], ids=["ahead", "between", "140 alike"])
def test_long_and_short_sequences_of_one_batch(hip, lens, dtype):
    """how many launches a long prompt takes is its own affair: every sequence comes out as in a call of its own"""
    import torch
    hk, hv, dk, dv = 8, 16, 64, 32
    rows, gate, beta, state = _inputs(17, lens, hk, hv, dk, dv, getattr(torch, dtype))
    got, new = _call(hip, rows, gate, beta, state, lens, hk, hv, dk, dv, True, 0.125)
    again, last = _call(hip, rows, gate, beta, state, lens, hk, hv, dk, dv, True, 0.125, in_place=True)
    assert torch.equal(got, again) and torch.equal(new, last)
    at = R.starts(lens)
    for i in sorted({0, 1, 5, 6, 7, len(lens) - 1}):
        one, st = _call(hip, rows[at[i]:at[i + 1]], gate[at[i]:at[i + 1]], beta[at[i]:at[i + 1]], state[i:i + 1], lens[i:i + 1], hk, hv, dk, dv, True, 0.125)
        assert torch.equal(got[at[i]:at[i + 1]], one) and torch.equal(new[i:i + 1], st), i
