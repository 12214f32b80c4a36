"""fm_logprobs_dev against 64 bits.

Tolerances.  d = x - m is off by half a step of |d|; e^d by that and a few steps, relatively, and sums
of them by a few more (at most 16 + 8 + 61 additions in a row): log Z by at most 96 half steps of fp32
absolutely, a log probability by 2 |log p| more.  The entropy adds sum p d, whose terms are off by
(|d| + 96) half steps of p |d|: at most 4 log(vocab)^2 in all, since sum p d^2 is at most
about log(vocab)^2 where the sum matters."""
import math

import pytest

from finchmoe_amd import binding as fb
from . import mix_ref as R

pytestmark = pytest.mark.gpu


def _call(hip, x, tokens, top_n, vocab=None):
    import torch
    rows, vocab = x.shape[0], vocab or x.shape[1]
    dx = x.cuda()
    dt = tokens.to(torch.int32).cuda()
    lp, en = torch.full((rows,), 99.0, device="cuda"), torch.full((rows,), 99.0, device="cuda")
    ids = torch.full((rows, max(top_n, 1)), -9, dtype=torch.int32, device="cuda")
    top = torch.full((rows, max(top_n, 1)), 99.0, device="cuda")
    torch.cuda.synchronize()
    hip.logprobs_dev(dx.data_ptr(), rows, vocab, x.shape[1], dt.data_ptr(), top_n, lp.data_ptr(), en.data_ptr(),
                     ids.data_ptr() if top_n else None, top.data_ptr() if top_n else None)
    hip.sync()
    return lp.cpu(), en.cpu(), ids[:, :top_n].cpu(), top[:, :top_n].cpu()


def _check(hip, x, tokens, top_n, vocab=None):
    import torch
    v = vocab or x.shape[1]
    lp, en, ids, top = R.logprobs(x[:, :v], tokens, top_n)
    g_lp, g_en, g_ids, g_top = _call(hip, x, tokens, top_n, vocab)
    fin = torch.isfinite(lp)
    assert torch.equal(g_lp[~fin].double(), lp[~fin])
    R.close(g_lp[fin], lp[fin], 96 * R.U24, 2 * R.U24, "log probability")
    R.close(g_en, en, R.U24 * (128 + 4 * math.log(max(v, 2)) ** 2), 0.0, "entropy")
    assert torch.equal(g_ids, ids)
    fin = torch.isfinite(top)
    assert torch.equal(g_top[~fin].double(), top[~fin])
    R.close(g_top[fin], top[fin], 96 * R.U24, 2 * R.U24, "top")


@pytest.mark.parametrize("top_n", [0, 1, 5, 20, 32])
@pytest.mark.parametrize("vocab", [32, 33, 1000, 4096, 4097, 8192, 50001, 248320])
def test_rows(hip, vocab, top_n):
    import torch
    g = torch.Generator().manual_seed(vocab + top_n)
    x = 3 * torch.randn(3, vocab, generator=g)
    x[1, 7] = 40.0                                         # one token takes all
    x[2] = 0.1 * torch.randn(vocab, generator=g)           # nearly uniform
    _check(hip, x, torch.tensor([0, 7, vocab - 1]), min(top_n, vocab))


@pytest.mark.parametrize("vocab", [1, 2, 5])
def test_tiny_vocabulary(hip, vocab):
    import torch
    _check(hip, torch.randn(4, vocab), torch.zeros(4, dtype=torch.int64), vocab)


def test_many_rows_strided(hip):
    import torch
    x = 2 * torch.randn(300, 5003)
    _check(hip, x, torch.arange(300) * 16, 7, vocab=4999)


@pytest.mark.parametrize("vocab", [100, 4096, 20000])
def test_ties_go_to_the_lowest_id(hip, vocab):
    import torch
    x = torch.zeros(4, vocab)
    x[1] = torch.randint(-2, 3, (vocab,)).float()
    x[2, ::2] = -0.0                                       # equal to +0
    x[3, vocab - 40:] = 1.0
    _check(hip, x, torch.tensor([5, 6, 7, vocab - 1]), 32)


def test_peaked_rows_keep_their_digits(hip):
    """entropies of 1e-3 and below, relative to their own size: Z' and sum e^d d are small sums, not
    differences (16 + 8 + 2 roundings of sums, a few of each term)"""
    import torch
    x = -20 + 0.5 * torch.randn(6, 9000)
    x[:, 4321] = torch.tensor([0.0, 2.0, 4.0, 8.0, 12.0, 20.0])
    tok = torch.full((6,), 4321)
    lp, en, _, _ = R.logprobs(x, tok, 0)
    g_lp, g_en, _, _ = _call(hip, x, tok, 0)
    # terms: |d| up to 40 half steps in e^d, sums and functions 64
    assert float(((g_lp.double() - lp) / lp).abs().max()) < 128 * R.U24
    assert float(((g_en.double() - en) / en).abs().max()) < 128 * R.U24


def test_masked_logits(hip):
    import torch
    x = torch.randn(5, 9000)
    x[0, 10:] = -float("inf")
    x[1, :] = -float("inf")
    x[2, ::3] = -float("inf")
    x[3, :4500] = -float("inf")
    x[4, 1:] = torch.finfo(torch.float32).min
    _check(hip, x, torch.tensor([10, 3, 1, 8999, 0]), 20)


def test_rows_of_nan_and_inf(hip):
    import torch
    x = torch.randn(4, 9000)
    x[1, 5000] = float("nan")
    x[2, 17] = float("inf")
    lp, en, ids, top = _call(hip, x, torch.tensor([1, 1, 1, 1]), 3)
    for r in (1, 2):
        assert math.isnan(lp[r]) and math.isnan(en[r]) and bool(torch.isnan(top[r]).all()) and ids[r].tolist() == [-1] * 3
    keep = [0, 3]
    _check(hip, x[keep], torch.tensor([1, 1]), 3)
    assert bool(torch.isfinite(lp[keep]).all())


def test_ids_outside_the_vocabulary(hip):
    import torch
    x = torch.randn(3, 500)
    lp, _, _, _ = _call(hip, x, torch.tensor([-1, 500, 2 ** 31 - 1]), 0)
    assert lp.tolist() == [-float("inf")] * 3


def test_outputs_are_optional_and_calls_repeat(hip):
    import torch
    x = torch.randn(2, 30000)
    full = _call(hip, x, torch.tensor([1, 2]), 4)
    dx, en = x.cuda(), torch.zeros(2, device="cuda")
    torch.cuda.synchronize()
    hip.logprobs_dev(dx.data_ptr(), 2, 30000, 30000, None, 0, None, en.data_ptr(), None, None)
    hip.sync()
    assert torch.equal(en.cpu(), full[1])
    for a, b in zip(full, _call(hip, x, torch.tensor([1, 2]), 4)):
        assert torch.equal(a, b)


def test_refusals(hip):
    import torch
    p = torch.zeros(4096, device="cuda").data_ptr()
    for args in ((None, 1, 100, 100, p, 0, p, p, None, None), (p, 0, 100, 100, p, 0, p, p, None, None),
                 (p, 1, 0, 100, p, 0, p, p, None, None), (p, 1, 100, 99, p, 0, p, p, None, None),
                 (p, 1, 100, 100, None, 0, p, p, None, None), (p, 1, 100, 100, p, 3, p, p, None, p),
                 (p, 1, 100, 100, p, 33, p, p, p, p), (p, 1, 10, 10, p, 11, p, p, p, p), (p, 1, 100, 100, p, 0, p, p, p, p),
                 (p + 2, 1, 100, 100, p, 0, p, p, None, None)):
        with pytest.raises(fb.FinchError) as e:
            hip.logprobs_dev(*args)
        assert e.value.status == fb.ERR_ARG


@pytest.mark.parametrize("stride", [5000, 5001])
def test_enough_rows_for_large_segments(hip, stride):
    """the form with more elements a thread, aligned rows and not, among them rows whose equal values are more
    than a segment collects"""
    import torch
    g = torch.Generator().manual_seed(stride)
    x = 2 * torch.randn(600, stride, generator=g)
    x[3] = 1.5
    x[4, :2500] = 7.0
    x[5] = -float("inf")
    x[6, 4999] = 60.0
    x[7] = torch.randint(0, 2, (stride,), generator=g).float()
    _check(hip, x, torch.arange(600) % 5000, 32, vocab=5000)
    bad = x[:600].clone()
    bad[9, 4000] = float("nan")
    lp, en, ids, top = _call(hip, bad, torch.zeros(600, dtype=torch.int64), 2, vocab=5000)
    assert math.isnan(lp[9]) and math.isnan(en[9]) and ids[9].tolist() == [-1, -1]
    assert bool(torch.isfinite(en[10:]).all())
