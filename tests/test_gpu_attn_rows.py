"""Attention over the 8-bit cache where an error counts for its own row: every element against its own bound
(tests/attn_rows.py), on narrow and wide tiles."""
import pytest

from . import attn_rows as A
from . import mix_ref as R
from .test_gpu_attn import Dev, _cache, _table

pytestmark = pytest.mark.gpu

DTYPES = ["float32", "bfloat16"]


def _run(hip, cache, table, lens, rows, q, scale, what=""):
    import torch
    ref, tol = A.attention(q, cache, table, lens, rows, scale, max(lens))
    got = Dev(hip, cache, table, lens).attn(q, rows, scale, max(lens))
    A.check(got, ref, tol, q.dtype, what)
    return got, ref


@pytest.mark.parametrize("rows", [[1] * 7, [30], [600]])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_bf16_calls_keep_the_weights(hip, d, rows):
    """few keys of nearly equal weight: with weights of 11 bits elements near the middle of two bf16 numbers go to the
    wrong one"""
    import torch
    lens, page = [5] * 7 if len(rows) > 1 else [5], 16
    g = torch.Generator().manual_seed(60 + d)
    cache, table = _cache(61, 8, 2, page, d), _table(62, lens, page, 8)
    q = (0.05 * torch.randn(sum(rows), 16, d, generator=g)).to(torch.bfloat16)
    _run(hip, cache, table, lens, rows, q, d ** -0.5)


def _paged(seed, d, rows, dtype, lead, value_scale, page=32, size=1.0):
    """Five pages; query head h and cache head 0 or 1 alike: dim 0 of a page's keys is +-127 and decides, `lead`
    (natural units) above or below; the rest is small noise.  value_scale: a factor a page."""
    import torch
    g = torch.Generator().manual_seed(seed)
    lens = [150] if len(rows) == 1 and rows[0] <= 150 else [rows[0]] if len(rows) == 1 else [150] * len(rows)
    n_pages = sum(-(-n // page) for n in lens) + 1
    cache, table = _cache(seed + 1, n_pages, 2, page, d), _table(seed + 2, lens, page, n_pages)
    cache[2].fill_(1.0 / 127)
    cache[0].copy_((torch.randn(cache[0].shape, generator=g) * 4).round().clamp(-12, 12).to(torch.int8))
    for s in range(len(lens)):
        for at in range(-(-lens[s] // page)):
            p = int(table[s, at])
            cache[0][p, :, :, 0] = int(127 * lead[at % len(lead)])
            cache[3][p] *= value_scale[at % len(value_scale)]
    q = 0.5 * torch.randn(sum(rows), 4, d, generator=g)
    q[:, :, 0] = 1.0
    return cache, table, lens, (q * size).to(getattr(torch, dtype))


ROWS = [[1], [1] * 9, [40], [600]]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", ROWS, ids=str)
@pytest.mark.parametrize("lead,values", [
    ((1, -1, 1, -1, 1), (1.0, 2.0 ** 60, 0.5, 2.0 ** 70, 3.0)),       # large values with next to no weight, between
    ((-1, -1, 1, 1, 1), (2.0 ** 60, 2.0 ** 65, 1.0, 0.3, 1.0)),       # ahead of the page that has the weight
    ((1, 1, -1, -1, -1), (2.0 ** -60, 2.0 ** -61, 2.0 ** 25, 1.0, 1.0)),      # behind it
    ((1, -1, 1, -1, 1), (1.0, 2.0 ** 115, 0.5, 2.0 ** 116, 3.0)),     # weight times value about alike
])
def test_values_count_by_their_weight(hip, lead, values, rows, dtype):
    """pages whose values are up to 2^116 apart, the smaller ones with (nearly) all of the weight: score 40 above and 40
    below, weights 2^115 apart"""
    cache, table, lens, q = _paged(70, 64, rows, dtype, lead, values)
    _run(hip, cache, table, lens, rows, q, 40.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", ROWS, ids=str)
@pytest.mark.parametrize("d", [64, 256])
def test_values_far_apart_with_like_weights(hip, d, rows, dtype):
    """small values count with the keys of their own row: rows that only see the small page keep its digits"""
    cache, table, lens, q = _paged(75, d, rows, dtype, (0.02, 0.0, -0.02, 0.01, 0.0), (1e-9, 1e-4, 300.0, 1e7, 1.0))
    _run(hip, cache, table, lens, rows, q, 1.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", ROWS, ids=str)
@pytest.mark.parametrize("power", [118, 103, -100, -115])
def test_values_near_the_ends_of_fp32(hip, power, rows, dtype):
    """values of up to 2^119 and down to 2^-121: a weighted mean of finite numbers is one"""
    f = 2.0 ** power
    cache, table, lens, q = _paged(80, 128, rows, dtype, (0.02, 0.0, -0.02, 0.01, 0.0), (f, 0.5 * f, f, 0.3 * f, 0.1 * f))
    _run(hip, cache, table, lens, rows, q, 1.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", ROWS, ids=str)
@pytest.mark.parametrize("power", [120, 110, -105, -120])
def test_queries_near_the_ends_of_fp32(hip, power, rows, dtype):
    cache, table, lens, q = _paged(85, 64, rows, dtype, (0.02, 0.0, -0.02, 0.01, 0.0), (1.0, 2.0), size=2.0 ** power)
    _run(hip, cache, table, lens, rows, q, 2.0 ** -power)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", ROWS, ids=str)
def test_large_scores(hip, rows, dtype):
    """scores in the thousands, where one key takes nearly all: every row against its own bound"""
    import torch
    lens, page, d = [max(rows[0], 100)] * len(rows), 16, 64
    n_pages = sum(-(-n // page) for n in lens) + 1
    cache, table = _cache(90, n_pages, 1, page, d), _table(91, lens, page, n_pages)
    g = torch.Generator().manual_seed(92)
    q = (torch.randn(sum(rows), 2, d, generator=g) * 300).to(getattr(torch, dtype))
    _run(hip, cache, table, lens, rows, q, 1.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_mixed_batches_with_values_far_apart(hip, dtype):
    """a prompt and single rows, the prompt's tiles split in parts, and long sequences joined from many parts"""
    rows = [200, 1, 1, 30]
    cache, table, lens, q = _paged(95, 128, rows, dtype, (1, -1, 0.9, -1, 1), (1.0, 2.0 ** 60, 0.5, 2.0 ** 70, 3.0))
    lens = [150] * 4
    _run(hip, cache, table, lens, rows, q, 40.0)
    import torch
    lens, rows, page, d = [2600], [3], 32, 64
    n_pages = 82
    cache, table = _cache(97, n_pages + 1, 2, page, d), _table(98, lens, page, n_pages)
    cache[3].mul_(torch.exp2(torch.randint(-30, 30, cache[3].shape, generator=torch.Generator().manual_seed(99)).float()))
    q = torch.randn(3, 4, d, generator=torch.Generator().manual_seed(100)).to(getattr(torch, dtype))
    _run(hip, cache, table, lens, rows, q, 6.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", ROWS, ids=str)
@pytest.mark.parametrize("score", [3e7, 3.1e7, -5e7, 1e8, 1.3e8, 1e20, -1e30])
def test_equal_scores_of_any_size(hip, score, rows, dtype):
    """keys of one and the same score have like weights, however large it is: the mean of the values seen.  Bound: the
    weights' own 8 half steps of fp32 and the sums', relative to the mean of |v|"""
    import torch
    page, d = 32, 128
    lens = [max(rows[0], 100)] * len(rows)
    n_pages = sum(-(-n // page) for n in lens) + 1
    cache, table = _cache(110, n_pages, 2, page, d), _table(111, lens, page, n_pages)
    cache[0].zero_()
    cache[0][..., 0] = 127
    cache[2].fill_(1.0 / 128)
    cache[3].fill_((1 - 2.0 ** -16) / 64)       # (just below a power of two)
    q = torch.randn(sum(rows), 4, d, generator=torch.Generator().manual_seed(112))
    q[..., 0] = 1.0
    q = q.to(getattr(torch, dtype))
    ref, _ = A.attention(q, cache, table, lens, rows, 0.0, max(lens))
    size = tuple(t.abs() if i in (1, 3) else t for i, t in enumerate(cache[:4])) + (page,)
    mean, _ = A.attention(q, size, table, lens, rows, 0.0, max(lens))
    got = Dev(hip, cache, table, lens).attn(q, rows, score, max(lens))
    A.check(got, ref, mean * (max(lens) / 32 + 48) * R.U24, q.dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [[1], [1] * 9, [600]], ids=str)
@pytest.mark.parametrize("page,lead", [(64, (1, -1, 1)), (64, (-1, 1, -1, 1, 1)), (128, (-1, 1, -1)), (16, (1, -1))])
def test_small_weights_of_large_values_are_joined(hip, page, lead, rows, dtype):
    """whole steps of keys 2^-121 the weight of the others, with values 2^121 their size: what one wave, half or part has
    counts as much as what another has.  Bound: one product a score, exact but for the scales' (three half steps), the
    difference and its shift (three more), twice; weights and sums as everywhere"""
    import math
    import torch
    d = 64
    lens = [max(rows[0], 64 * 5)] * len(rows)
    n_pages = sum(-(-n // page) for n in lens) + 1
    cache, table = _cache(120, n_pages, 2, page, d), _table(121, lens, page, n_pages)
    cache[0].zero_()
    cache[2].fill_(1.0 / 127)
    for s in range(len(lens)):
        for at in range(-(-lens[s] // page)):
            p = int(table[s, at])
            cache[0][p, :, :, 0] = 127 * lead[at % len(lead)]
            cache[3][p] = (1.0 + 0.1 * (at % 7)) * (2.0 ** 119 if lead[at % len(lead)] < 0 else 0.25)
    q = torch.randn(sum(rows), 4, d, generator=torch.Generator().manual_seed(122))
    q[..., 0] = 1.0
    q = q.to(getattr(torch, dtype))
    ref, _ = A.attention(q, cache, table, lens, rows, 42.0, max(lens))
    size = tuple(t.abs() if i in (1, 3) else t for i, t in enumerate(cache[:4])) + (page,)
    of_size, _ = A.attention(q, size, table, lens, rows, 42.0, max(lens))
    got = Dev(hip, cache, table, lens).attn(q, rows, 42.0, max(lens))
    A.check(got, ref, of_size * (math.expm1(2 * 6 * 42 * R.U24) + (max(lens) / 32 + 48) * R.U24), q.dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,rows", [([20011], [1]), ([40000, 3], [3, 1])], ids=["20011", "40000 and 3"])
def test_more_parts_than_a_wave_has_lanes(hip, lens, rows, dtype):
    """a row's keys over 79 and 157 workgroups, values of pages 2^40 apart"""
    import torch
    page, d = 128, 64
    n_pages = sum(-(-n // page) for n in lens) + 1
    g = torch.Generator().manual_seed(130)
    cache, table = _cache(131, n_pages, 1, page, d), _table(132, lens, page, n_pages)
    cache[3].mul_(torch.exp2(torch.randint(-20, 20, cache[3].shape, generator=g).float()))
    q = (1.5 * torch.randn(sum(rows), 2, d, generator=g)).to(getattr(torch, dtype))
    _run(hip, cache, table, lens, rows, q, 0.125)
