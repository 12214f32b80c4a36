"""The 8-bit paged cache and its attention (fm_kv_append_dev, fm_kv_read_dev, fm_attn_dev) against
64-bit forms.

What the cache holds is compared exactly: codes are rounded quotients, scales one fp32 product with 1/127.

Tolerance of attention.  With A the largest scale * sum |q_i k_i| of a visible pair and V the
largest |v|: fp32 queries keep 22 bits of a row's largest element and the sums over head_dim round
in fp32, so a score is off by at most A (head_dim + 8) 2^-24; weights of a softmax move by at most twice
that, relatively, and so does the output, in units of V.  The weights themselves keep 22 bits
(fp32: 8 half steps of fp32 with exp2's own) or 11 (bf16: 2^-11), and sums over N keys run
32 at a time with at most N / 32 + 40 roundings.  bf16 outputs add half a step of bf16."""
import numpy as np
import pytest

from finchmoe_amd import binding as fb
from . import mix_ref as R

pytestmark = pytest.mark.gpu


def _cache(seed, n_pages, kv, page, d):
    import torch
    g = torch.Generator().manual_seed(seed)
    codes = lambda *s: (torch.randn(*s, generator=g) * 40).clamp(-127, 127).round().to(torch.int8)  # noqa: E731
    return (codes(n_pages, kv, page, d), codes(n_pages, kv, d, page), 0.005 + 0.02 * torch.rand(n_pages, kv, generator=g),
            0.005 + 0.02 * torch.rand(n_pages, kv, generator=g), page)


def _table(seed, lens, page, n_pages, more=0):
    import torch
    g = torch.Generator().manual_seed(seed)
    per = [-(-n // page) for n in lens]
    order = torch.randperm(n_pages, generator=g).to(torch.int32)
    t = torch.full((len(lens), max(max(per), 1) + more), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(per):
        t[s, :n] = order[at:at + n]
        at += n
    assert at <= n_pages
    return t


class Dev:
    """the cache and its table on the device"""

    def __init__(self, hip, cache, table, lens):
        import torch
        self.hip = hip
        self.k, self.v, self.ks, self.vs = (t.cuda() for t in cache[:4])
        self.page, self.table = cache[4], table.cuda()
        self.len = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.n_seq = len(lens)

    def desc(self):
        n, kv, page, d = self.k.shape
        return self.hip.kv_cache(d_k=self.k.data_ptr(), d_v=self.v.data_ptr(), d_k_scale=self.ks.data_ptr(),
                                 d_v_scale=self.vs.data_ptr(), n_pages=n, page_tokens=page, kv_heads=kv, head_dim=d)

    def attn_args(self, q, rows, scale, max_len, out, one_row=False, q_stride=None):
        import torch
        return self.hip.attn_args(
            cache=self.desc(), n_seq=self.n_seq, q_heads=out.shape[1], scale=scale, d_q=q.data_ptr(),
            dtype=fb.DTYPE_BF16 if q.dtype == torch.bfloat16 else fb.DTYPE_F32, q_stride=q_stride,
            seq_start=None if one_row else R.starts(rows), d_len=self.len.data_ptr(), d_pages=self.table.data_ptr(),
            max_pages=self.table.shape[1], max_len=max_len, d_out=out.data_ptr())

    def attn(self, q, rows, scale, max_len, **kw):
        import torch
        q = q.cuda()
        out = torch.full(q.shape, float("nan"), dtype=q.dtype, device="cuda")
        torch.cuda.synchronize()
        self.hip.attn_dev(self.attn_args(q, rows, scale, max_len, out, **kw))
        self.hip.sync()
        return out.float().cpu()

    def rows(self, fn, k, v, rows, strides=(None, None)):
        import torch
        torch.cuda.synchronize()
        fn(self.hip.kv_args(cache=self.desc(), n_seq=self.n_seq, d_k=k.data_ptr(), d_v=v.data_ptr(), k_stride=strides[0],
                            v_stride=strides[1], dtype=fb.DTYPE_BF16 if k.dtype == torch.bfloat16 else fb.DTYPE_F32,
                            seq_start=R.starts(rows), d_len=self.len.data_ptr(), d_pages=self.table.data_ptr(),
                            max_pages=self.table.shape[1]))
        self.hip.sync()


def _tol(most, vmax, d, n, bf):
    return vmax * (2 * most * (d + 8) * R.U24 + (2.0 ** -11 if bf else 8 * R.U24) + (n / 32 + 40) * R.U24)


def _run(hip, seed, lens, rows, hq, kv, d, page, dtype, max_len=None, more=0, spoil=None, **kw):
    import torch
    n_pages = sum(-(-n // page) for n in lens) + 2
    cache = _cache(seed, n_pages, kv, page, d)
    table = _table(seed + 1, lens, page, n_pages, more)
    if spoil:
        spoil(cache, table)
    g = torch.Generator().manual_seed(seed + 2)
    q = (1.5 * torch.randn(sum(rows), hq, d, generator=g)).to(getattr(torch, dtype))
    max_len = max_len or max(max(lens), 1)
    scale = d ** -0.5
    ref, most, vmax = R.attention(q, cache, table, lens, rows, scale, max_len)
    got = Dev(hip, cache, table, lens).attn(q, rows, scale, max_len, **kw)
    bf = dtype == "bfloat16"
    R.close(got, ref, _tol(most, vmax, d, max(lens), bf), R.U_BF16 if bf else 0.0, "lens %s rows %s" % (lens, rows))
    return got, ref


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_one_row_per_sequence(hip, page, d, dtype):
    _run(hip, page + d, [1, 15, 64, 65, 300], [1] * 5, 4, 2, d, page, dtype, one_row=True)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("hq,kv", [(1, 1), (3, 1), (16, 1), (20, 1), (8, 4), (6, 2)])
def test_head_layouts(hip, hq, kv, dtype):
    _run(hip, hq * 10 + kv, [77, 130], [1, 1], hq, kv, 64, 32, dtype)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("d,hq,kv", [(64, 4, 1), (128, 4, 2), (256, 2, 1), (128, 7, 1)])
@pytest.mark.parametrize("lens,rows", [([40], [40]), ([130], [130]), ([200], [33]), ([9, 70, 150], [2, 70, 17]),
                                       ([90, 5, 64], [64, 0, 65])])
def test_several_rows(hip, lens, rows, d, hq, kv, dtype):
    """causal rows, ragged, an empty sequence, and one with more rows than tokens"""
    _run(hip, sum(lens) + d, lens, rows, hq, kv, d, 16, dtype)


@pytest.mark.parametrize("rows", [[1], [3], [24]])
def test_long_context_in_chunks(hip, rows):
    """many workgroups over the keys, the last chunk short"""
    _run(hip, 5, [5003], rows, 4, 2, 64, 64, "float32")
    _run(hip, 6, [5003], rows, 4, 2, 64, 64, "bfloat16")


@pytest.mark.parametrize("rows", [[1] * 30, [300]])
def test_fp32_weights_keep_their_second_piece(hip, rows):
    """many columns, page scales of their own: no single weight may drop to 11 bits (an error of 2^-12 of
    it, far above the bound, in one row of thousands)"""
    lens = [300] if len(rows) == 1 else [40 + 7 * i for i in range(30)]
    for seed in (50, 51):
        _run(hip, seed, lens, rows, 8, 2, 128, 64, "float32")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 128), (256, 32)])
@pytest.mark.parametrize("lens,rows", [([140, 1, 300, 0, 33], [140, 1, 70, 0, 5]), ([700], [200]), ([260] * 5, [9, 40, 3, 60, 41])])
def test_both_tile_widths_in_one_batch(hip, lens, rows, d, page, dtype):
    """enough columns for wide tiles beside sequences that keep narrow ones; wide tiles split in parts"""
    _run(hip, sum(rows) + d, lens, rows, 8, 2, d, page, dtype)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 128), (256, 32)])
@pytest.mark.parametrize("lens,rows", [([140, 1, 300, 0, 33], [140, 1, 70, 0, 5]), ([900, 260, 5], [130, 1, 5])])
def test_both_tile_widths_where_lengths_may_grow(hip, lens, rows, d, page, dtype):
    """a bound of the lengths far above them: short sequences keep narrow tiles beside the wide ones"""
    _run(hip, sum(rows) + d + 1, lens, rows, 8, 2, d, page, dtype, max_len=40000, more=40000 // page)


def test_ragged_lengths_share_one_cut(hip):
    _run(hip, 7, [3, 4000, 700], [1, 1, 1], 2, 1, 64, 16, "float32")


def test_rows_that_see_nothing(hip):
    import torch
    lens, rows = [0, 20, 4], [1, 1, 6]
    got, ref = _run(hip, 8, lens, rows, 2, 1, 64, 16, "float32")
    assert float(got[0].abs().max()) == 0.0
    assert float(got[2:4].abs().max()) == 0.0 and float(got[4:].abs().amax(-1).min()) > 0.0


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows", [[1, 1], [40, 90], [300, 90]])
def test_pages_that_are_not_there(hip, rows, dtype):
    """entries outside the pool are not seen; a sequence with none left gives zeros"""
    def spoil(cache, table):
        table[0, :] = -1
        table[1, 1] = cache[0].shape[0]
        table[1, 3] = -7
    got, _ = _run(hip, 9, [40, 130], rows, 4, 2, 64, 32, dtype, spoil=spoil)
    assert float(got[:rows[0]].abs().max()) == 0.0


@pytest.mark.parametrize("rows", [[1], [30], [530]])
def test_shorter_max_len_and_table(hip, rows):
    _run(hip, 10, [200], rows, 2, 1, 64, 32, "float32", max_len=190)
    # more tokens than the table has pages for
    import torch
    page, lens = 32, [100]
    cache = _cache(11, 8, 1, page, 64)
    table = torch.tensor([[3, 5]], dtype=torch.int32)
    q = torch.randn(sum(rows), 2, 64)
    ref, most, vmax = R.attention(q, cache, table, lens, rows, 0.1, 100)
    got = Dev(hip, cache, table, lens).attn(q, rows, 0.1, 100)
    R.close(got, ref, _tol(most, vmax, 64, 64, False), 0.0, "short table")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows", [[1], [20], [530]])
def test_what_is_masked_may_be_anything(hip, rows, dtype):
    """scales of pages behind the length are NaN and inf, so are later pages of the pool"""
    def spoil(cache, table):
        used = set(table[0, :3].tolist())
        for p in range(cache[0].shape[0]):
            if p not in used:
                cache[2][p] = float("nan")
                cache[3][p] = float("inf")
        table[0, 3:] = torch_int(cache[0].shape[0] - 1)
    def torch_int(v):
        return v
    _run(hip, 12, [70], rows, 2, 1, 64, 32, dtype, more=4, spoil=spoil, max_len=200)


@pytest.mark.parametrize("rows", [[1], [40], [530]])
def test_value_scales_of_very_different_size(hip, rows):
    """pages whose values are 10^4 apart, in either order, and large ones"""
    def spoil(cache, table):
        for at, f in enumerate((1e-4, 300.0, 1.0, 1e4, 1e-3)):
            cache[3][int(table[0, at])] *= f
    _run(hip, 13, [150], rows, 2, 1, 128, 32, "float32", spoil=spoil)
    _run(hip, 13, [150], rows, 2, 1, 128, 32, "bfloat16", spoil=spoil)


@pytest.mark.parametrize("size", [1e-30, 1e-3, 1e3])
@pytest.mark.parametrize("rows", [[1], [40], [530]])
def test_queries_of_any_size(hip, rows, size):
    import torch
    lens, page, d = [100], 16, 64
    cache, table = _cache(14, 8, 1, page, d), _table(15, lens, page, 8)
    q = torch.randn(sum(rows), 2, d) * size
    scale = 0.125 / max(size, 1e-30)
    ref, most, vmax = R.attention(q, cache, table, lens, rows, scale, 100)
    got = Dev(hip, cache, table, lens).attn(q, rows, scale, 100)
    R.close(got, ref, _tol(most, vmax, d, 100, False), 0.0, "size %g" % size)


@pytest.mark.parametrize("rows", [[1], [40], [530]])
def test_large_scores_and_nan_rows(hip, rows):
    """scores in the thousands (one key takes all), and a query of NaN poisons its own row and head alone"""
    import torch
    lens, page, d = [100], 16, 64
    cache, table = _cache(16, 8, 1, page, d), _table(17, lens, page, 8)
    q = torch.randn(sum(rows), 2, d) * 300
    ref, _, vmax = R.attention(q, cache, table, lens, rows, 1.0, 100)
    q[-1, 1, 3] = float("nan")          # (the last row sees every key)
    got = Dev(hip, cache, table, lens).attn(q, rows, 1.0, 100)
    assert bool(torch.isnan(got[-1, 1]).all())
    fine = torch.ones(q.shape[:2], dtype=torch.bool)
    fine[-1, 1] = False
    assert bool(torch.isfinite(got[fine]).all())
    # (two nearly equal scores of a thousand may share the weight differently: none here)
    near = (got[fine].double() - ref[fine]).abs().amax(-1)      # (rows that see nothing: zeros in both)
    assert float(near.median()) <= vmax * 1e-3


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows", [[40, 1], [300, 1]])
def test_strided_queries(hip, rows, dtype):
    import torch
    lens, page, d, hq = [90, 33], 32, 64, 4
    n = sum(rows)
    cache, table = _cache(18, 8, 2, page, d), _table(19, lens, page, 8)
    wide = torch.randn(n, hq * d + 24).to(getattr(torch, dtype)).cuda()
    q = wide[:, 8:8 + hq * d]
    ref, most, vmax = R.attention(q.cpu().reshape(n, hq, d), cache, table, lens, rows, 0.125, 90)
    dev = Dev(hip, cache, table, lens)
    out = torch.empty(n, hq, d, dtype=wide.dtype, device="cuda")
    torch.cuda.synchronize()
    hip.attn_dev(dev.attn_args(q, rows, 0.125, 90, out, q_stride=wide.shape[1]))
    hip.sync()
    bf = dtype == "bfloat16"
    R.close(out, ref, _tol(most, vmax, d, 90, bf), R.U_BF16 if bf else 0.0, "strided")


@pytest.mark.parametrize("rows", [[1, 1, 1], [3, 90, 20], [3, 180, 20]])
def test_attention_repeats_bit_for_bit(hip, rows):
    import torch
    lens, page, d = [3000, 100, 700], 32, 128
    cache, table = _cache(20, 140, 2, page, d), _table(21, lens, page, 140)
    dev = Dev(hip, cache, table, lens)
    q = torch.randn(sum(rows), 6, d)
    a = dev.attn(q, rows, 0.1, 3000)
    for _ in range(3):
        assert torch.equal(a, dev.attn(q, rows, 0.1, 3000))


# ---- the cache ---------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("kv,d,page", [(1, 64, 16), (2, 128, 32), (3, 256, 64), (1, 64, 128)])
@pytest.mark.parametrize("lens,rows", [([1], [1]), ([50], [50]), ([130, 64, 7], [3, 64, 0]), ([200], [37]), ([5, 3], [9, 1])])
def test_append_and_read(hip, lens, rows, kv, d, page, dtype):
    """codes and scales exactly; everything else of the pool as it was"""
    import torch
    dt = getattr(torch, dtype)
    n_pages = sum(-(-n // page) for n in lens) + 3
    cache = _cache(sum(lens) + d, n_pages, kv, page, d)
    table = _table(1, lens, page, n_pages, more=1)
    g = torch.Generator().manual_seed(2)
    size = torch.exp(1.5 * torch.randn(sum(rows), 1, 1, generator=g))
    k = (torch.randn(sum(rows), kv, d, generator=g) * size).to(dt)
    v = (torch.randn(sum(rows), kv, d, generator=g) * 0.3).to(dt)
    want = R.append(cache, table, lens, rows, k, v)
    dev = Dev(hip, cache, table, lens)
    dk, dv = k.cuda(), v.cuda()
    for _ in range(2):      # the same rows again change nothing
        dev.rows(hip.kv_append_dev, dk, dv, rows)
        for name, got, ref in zip(("k", "v", "k scale", "v scale"), (dev.k, dev.v, dev.ks, dev.vs), want):
            assert torch.equal(got.cpu(), ref), name
    back = [min(n, page * table.shape[1]) for n in lens]
    ko = torch.full((sum(back), kv, d), float("nan"), device="cuda")
    vo = torch.full_like(ko, float("nan"))
    dev.rows(hip.kv_read_dev, ko, vo, back)
    at = R.starts(back)
    for s, n in enumerate(back):
        rk, rv, _ = R.page_values(*want, table[s], n, page)
        assert torch.equal(ko[at[s]:at[s + 1]].cpu(), rk.float()) and torch.equal(vo[at[s]:at[s + 1]].cpu(), rv.float())


def test_append_token_by_token(hip):
    """a growing sequence: scales only grow, old codes are rounded to each new one"""
    import torch
    kv, d, page = 2, 64, 16
    cache = _cache(30, 4, kv, page, d)
    table = torch.tensor([[2, 0]], dtype=torch.int32)
    g = torch.Generator().manual_seed(31)
    dev = Dev(hip, cache, table, [0])
    ref = cache
    for n in range(1, 21):
        k, v = torch.randn(1, kv, d, generator=g) * n, torch.randn(1, kv, d, generator=g) / n
        ref = R.append(ref, table, [n], [1], k, v) + (page,)
        dev.len.fill_(n)
        dev.rows(hip.kv_append_dev, k.cuda(), v.cuda(), [1])
        for got, want in zip((dev.k, dev.v, dev.ks, dev.vs), ref[:4]):
            assert torch.equal(got.cpu(), want), n


def test_append_values_on_the_border(hip):
    """quotients half-way between two codes go to the even one; neighbours in fp32 do not"""
    import torch
    page, d = 16, 64
    cache = _cache(32, 2, 1, page, d)
    table = torch.tensor([[0]], dtype=torch.int32)
    k = torch.zeros(16, 1, d)
    k[0, 0, 0] = 127.0                                    # scale 1
    half = torch.arange(-126, 126).float() + 0.5
    k.view(-1)[1:1 + half.numel()] = half
    k.view(-1)[300:300 + half.numel()] = torch.nextafter(half, torch.full_like(half, 1e9))
    k.view(-1)[600:600 + half.numel()] = torch.nextafter(half, torch.full_like(half, -1e9))
    v = k * 0.37
    want = R.append(cache, table, [16], [16], k, v)
    dev = Dev(hip, cache, table, [16])
    dev.rows(hip.kv_append_dev, k.cuda(), v.cuda(), [16])
    assert torch.equal(dev.k.cpu(), want[0]) and torch.equal(dev.v.cpu(), want[1]) and torch.equal(dev.vs.cpu(), want[3])


def test_append_infinities_nan_and_zeros(hip):
    import torch
    page, d = 16, 64
    cache = _cache(33, 3, 2, page, d)
    table = torch.tensor([[1]], dtype=torch.int32)
    k = torch.randn(5, 2, d)
    k[0, 0, 0], k[1, 0, 1], k[2, 0, 2] = float("inf"), -float("inf"), float("nan")
    k[:, 1] = 0.0
    v = torch.full((5, 2, d), float("nan"))
    v[0, 1, 0] = float("inf")
    want = R.append(cache, table, [5], [5], k, v)
    dev = Dev(hip, cache, table, [5])
    dev.rows(hip.kv_append_dev, k.cuda(), v.cuda(), [5])
    for got, ref in zip((dev.k, dev.v, dev.ks, dev.vs), want):
        assert torch.equal(got.cpu(), ref)
    assert float(dev.ks[1, 1]) == 0.0 and float(dev.vs[1].abs().max()) == 0.0


def test_append_to_pages_that_are_not_there(hip):
    """nothing is written, also not behind the table's end; reading gives zeros"""
    import torch
    page, d = 16, 64
    cache = _cache(34, 4, 1, page, d)
    table = torch.tensor([[9, 1], [-1, 2]], dtype=torch.int32)
    lens, rows = [50, 30], [50, 30]
    k, v = torch.randn(80, 1, d), torch.randn(80, 1, d)
    want = R.append(cache, table, lens, rows, k, v)
    dev = Dev(hip, cache, table, lens)
    dev.rows(hip.kv_append_dev, k.cuda(), v.cuda(), rows)
    for got, ref in zip((dev.k, dev.v, dev.ks, dev.vs), want):
        assert torch.equal(got.cpu(), ref)
    ko, vo = torch.full((80, 1, d), 7.0, device="cuda"), torch.full((80, 1, d), 7.0, device="cuda")
    dev.rows(hip.kv_read_dev, ko, vo, rows)
    assert float(ko[:16].abs().max()) == 0.0 and float(vo[32:50].abs().max()) == 0.0 and float(ko[50:66].abs().max()) == 0.0
    assert float(ko[16:32].abs().min(-1).values.max()) > 0.0


def test_strided_rows(hip):
    import torch
    page, d, kv, lens = 32, 64, 2, [45]
    cache, table = _cache(35, 3, kv, page, d), _table(36, [45], page, 3)
    wide = torch.randn(45, 3 * kv * d)
    k, v = wide[:, :kv * d], wide[:, kv * d:2 * kv * d]
    want = R.append(cache, table, lens, lens, k.reshape(45, kv, d), v.reshape(45, kv, d))
    dev = Dev(hip, cache, table, lens)
    dw = wide.cuda()
    dev.rows(hip.kv_append_dev, dw[:, :kv * d], dw[:, kv * d:2 * kv * d], lens, strides=(3 * kv * d,) * 2)
    assert torch.equal(dev.k.cpu(), want[0]) and torch.equal(dev.v.cpu(), want[1])


def test_offsets_past_32_bits(hip):
    """a pool of more than 4 GiB of codes: the last pages are written, read and attended to"""
    import torch
    page, d, kv = 128, 256, 4
    n_pages = (1 << 32) // (page * d * kv) + 8
    k = torch.zeros(n_pages, kv, page, d, dtype=torch.int8, device="cuda")
    v = torch.zeros(n_pages, kv, d, page, dtype=torch.int8, device="cuda")
    ks, vs = torch.ones(n_pages, kv, device="cuda"), torch.ones(n_pages, kv, device="cuda")
    table = torch.tensor([[n_pages - 1, 0, n_pages - 2]], dtype=torch.int32)
    lens = [300]
    g = torch.Generator().manual_seed(40)
    x, y = torch.randn(300, kv, d, generator=g), torch.randn(300, kv, d, generator=g)
    dev = Dev(hip, (k[:1], v[:1], ks, vs, page), table, lens)
    dev.k, dev.v = k, v
    dev.rows(hip.kv_append_dev, x.cuda(), y.cuda(), lens)
    pick = [n_pages - 1, 0, n_pages - 2]
    small = tuple(t[pick].cpu() for t in (dev.k, dev.v, dev.ks, dev.vs)) + (page,)
    want = R.append((torch.zeros_like(small[0]), torch.zeros_like(small[1]), torch.ones(3, kv), torch.ones(3, kv), page),
                    torch.tensor([[0, 1, 2]]), lens, lens, x, y)
    for got, ref in zip(small, want):
        assert torch.equal(got, ref)
    for rows in ([1], [50], [270]):
        q = torch.randn(sum(rows), kv, d, generator=g)
        ref, most, vmax = R.attention(q, small, torch.tensor([[0, 1, 2]]), lens, rows, 0.1, 300)
        R.close(dev.attn(q, rows, 0.1, 300), ref, _tol(most, vmax, d, 300, False), 0.0, "far pages")


def test_refusals(hip):
    import torch
    z = torch.zeros(1 << 16, device="cuda")
    p = z.data_ptr()
    shape = dict(n_pages=2, page_tokens=16, kv_heads=1, head_dim=64)
    good = dict(n_seq=1, q_heads=1, d_q=p, d_len=p, d_pages=p, max_pages=1, max_len=16, d_out=p + 4096, scale=1.0)

    def status(cache=None, **kw):
        c = hip.kv_cache(**dict(dict(d_k=p, d_v=p, d_k_scale=p, d_v_scale=p), **dict(shape, **(cache or {}))))
        with pytest.raises(fb.FinchError) as e:
            hip.attn_dev(hip.attn_args(cache=c, **dict(good, **kw)))
        return e.value.status

    assert status({"page_tokens": 48}) == fb.ERR_UNSUPPORTED and status({"head_dim": 96}) == fb.ERR_UNSUPPORTED
    assert status({"d_k": p + 8}) == fb.ERR_ARG and status({"n_pages": 0}) == fb.ERR_ARG
    assert status({"kv_heads": 2}, q_heads=3) == fb.ERR_ARG and status(q_stride=60) == fb.ERR_ARG
    assert status(max_len=-1) == fb.ERR_ARG and status(n_seq=0) == fb.ERR_ARG and status(n_seq=257) == fb.ERR_ARG
    assert status(seq_start=[1, 2]) == fb.ERR_ARG and status(d_len=None) == fb.ERR_ARG
    c = hip.kv_cache(d_k=p, d_v=p, d_k_scale=p, d_v_scale=p, **shape)
    with pytest.raises(fb.FinchError):
        hip.kv_read_dev(hip.kv_args(cache=c, n_seq=1, d_k=p, d_v=p, d_len=p, d_pages=p, max_pages=1, dtype=fb.DTYPE_BF16))
