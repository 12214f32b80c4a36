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
