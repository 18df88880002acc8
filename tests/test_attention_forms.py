"""kv_cache_attention in each of its forms (tiles of 16, 32 and 128 rows, contexts whole and cut), every test saying which form it runs."""

import ctypes
import itertools
import math

import pytest
import torch

from oracle import decoder_reference as R
from tilegym_amd import _lib, ops

from .test_decoder_ops import BF16, F16, HALF, Pool


def form_of(tokens, q_heads, batch, kv_heads, dim, page, width, window=0, sinks=0):
    """(rows of a tile, parts that contexts are cut into)."""
    out = (ctypes.c_int32 * 2)()
    assert _lib.load().tg_diag_kv_attention_form(tokens, q_heads, batch, kv_heads, dim, page, width, window, sinks, out) == 0
    return tuple(out)


def test_form_query_needs_no_device():
    out = (ctypes.c_int32 * 2)()
    query = _lib.load().tg_diag_kv_attention_form
    assert query(0, 4, 1, 1, 64, 16, 1, 0, 0, out) == -6 and query(1, 4, 1, 3, 64, 16, 1, 0, 0, out) == -6 and query(1, 4, 1, 1, 64, 16, 1, -1, 0, out) == -6
    assert query(2 ** 62, 4, 1, 1, 64, 16, 1, 0, 0, out) == -6
    assert query(1, 4, 1, 1, 64, 16, 1, 0, 0, None) == -5
    assert form_of(1, 4, 1, 1, 64, 16, 1) == (16, 1)
    # cut exactly where there is scratch memory to be had
    need = _lib.load().tg_fp8_kv_attention_workspace_bytes
    for sizes in itertools.product((1, 40, 600), (8, 32), (1, 9), (8,), (64, 128, 256), (16, 128), (1, 30), (0, 500), (0,)):
        assert (form_of(*sizes)[1] > 1) == (need(*sizes) > 0), sizes


def test_oracle_by_head_agrees():
    g = torch.Generator().manual_seed(2)
    lens, indptr = [9, 3, 40], [0, 4, 9, 11]  # (sequence 1 has fewer tokens than new ones)
    k, v = ([torch.randn(n, 2, 64, generator=g, dtype=torch.float64) for n in lens] for _ in range(2))
    q = torch.randn(11, 6, 64, generator=g)
    for window, sinks in ((0, 0), (3, 0), (5, 2)):
        a, tol = R.ref_attention(q, k, v, lens, indptr, 0.2, window, sinks, 2.0 ** -8)
        b, tol2 = R.ref_attention_by_head(q, k, v, lens, indptr, 0.2, window, sinks, 2.0 ** -8)
        assert bool(((a - b).abs() <= 1e-12).all()) and bool(((tol - tol2).abs() <= 1e-3 * tol + 1e-12).all())


class Forms(Pool):
    """A pool whose tables list pages in turn, with the scale of every position."""

    def scales(self, lens):
        s = self.cache.v_scale.double()
        return [torch.cat([s[p][None].expand(self.page, -1) if 0 <= p < s.shape[0] else torch.ones(self.page, s.shape[1], dtype=torch.float64, device=s.device)
                           for p in self.table[b]])[:n] for b, n in enumerate(lens)]

    def rows(self, name, lens):
        """Of the positions that the table has; pages that are not there are zeros (no token sees them)."""
        return [x.nan_to_num(0.0).to(self.device) for x in super().rows(name, lens)]

    def queries(self, tokens, heads, dtype, factor=1.0):
        wide = torch.randn(tokens, heads + 3, self.dim, generator=self.g) * factor
        return wide.to(dtype).to(self.device)[:, 2:2 + heads]

    def attend(self, q, lens, news, window=0, sinks=0, sm_scale=None, table=None):
        indptr = [0] + list(itertools.accumulate(news))
        got = ops.kv_cache_attention(q, self.cache, self.i32(table or self.table), self.i32(lens), self.i32(indptr), sm_scale=sm_scale, window=window,
                                     sink_tokens=sinks)
        return got, indptr

    def check(self, q, lens, news, window=0, sinks=0, sm_scale=None, table=None):
        got, indptr = self.attend(q, lens, news, window, sinks, sm_scale, table)
        scale = self.dim ** -0.5 if sm_scale is None else sm_scale
        want, tol = R.ref_attention_by_head(q, self.rows("k", lens), self.rows("v", lens), lens, indptr, scale, window, sinks, HALF[q.dtype], self.scales(lens))
        err = (got.double() - want).abs()
        assert bool((err <= tol).all()), (float((err / tol).nan_to_num(math.inf).max()), lens, news, window, sinks)
        return got


# (rows of a tile, whether contexts are cut): heads, query heads to each, head dims, (lengths, new tokens)
FORMS = {
    (16, False): (2, 4, (64, 128, 256), ([1000, 90, 700], [3, 5, 1])),
    (16, True): (2, 4, (64, 128, 256), ([1900, 90, 700], [3, 5, 1])),
    (32, False): (2, 5, (64, 128), ([1000, 130], [150, 30])),
    (32, True): (2, 5, (64, 128), ([1900, 130], [150, 30])),
    (128, False): (8, 4, (64, 128, 256), ([1000, 90], [281, 40])),
    (128, True): (8, 4, (64, 128, 256), ([1900, 90], [281, 40])),
}
CASES = [(form, dim) for form, (_, _, dims, _) in FORMS.items() for dim in dims]


def _pool_of(device, form, dim, page, dtype):
    heads, group, _, (lens, news) = FORMS[form]
    width = -(-max(lens) // page)
    pool = Forms(device, width * len(lens), heads, page, dim, len(lens), width, seed=dim + page)
    pool.fill(lens, lens, dtype)
    return pool, group, lens, news, width


@pytest.mark.gpu
@pytest.mark.parametrize("form,dim", CASES)
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_form(device, form, dim, page, dtype):
    """Many steps of keys; then a window with first tokens, whose unseen pages are not there."""
    pool, group, lens, news, width = _pool_of(device, form, dim, page, dtype)
    heads = pool.heads * group
    q = pool.queries(sum(news), heads, dtype, 3.0)
    for window, sinks in ((0, 0), (950 if form[1] else 300, 70), (33, 0)):
        rows, parts = form_of(sum(news), heads, len(lens), pool.heads, dim, page, width, window, sinks)
        assert rows == form[0] and (parts > 1) == (form[1] and window != 33)
        table = [row[:] for row in pool.table]
        if window:
            for b, (length, n) in enumerate(zip(lens, news)):
                first = max(0, length - n - window + 1)
                for i in range(width):
                    if i * page >= length or (i * page >= sinks and (i + 1) * page <= first):
                        table[b][i] = -1 if i % 2 else 10 ** 6
        pool.check(q, lens, news, window, sinks, table=table)
    pool.check(q, lens, news, sm_scale=-0.2)


def test_sizes_reach_the_forms():
    for form, dim in CASES:
        heads, group, _, (lens, news) = FORMS[form]
        for page in (16, 32, 64, 128):
            sizes = (sum(news), heads * group, len(lens), heads, dim, page, -(-max(lens) // page))
            assert form_of(*sizes)[0] == form[0] and (form_of(*sizes)[1] > 1) == form[1], (form, dim, page)


@pytest.mark.gpu
@pytest.mark.parametrize("form,dim", CASES)
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_rows_that_are_no_numbers_show_it(device, form, dim, page, dtype):
    """A NaN in q, an infinity, and (bf16) one key whose score overflows: those rows come out as no numbers whether contexts are cut or
    not, and the other rows as ever."""
    pool, group, lens, news, width = _pool_of(device, form, dim, page, dtype)
    heads, total = pool.heads * group, sum(news)
    assert form_of(total, heads, len(lens), pool.heads, dim, page, width)[0] == form[0]
    key = 700 if form[1] else 70  # (in one part of a cut context)
    pool.cache.k.view(torch.uint8)[:, :, :, 0] = 0
    pool.cache.k.view(torch.uint8)[pool.table[0][key // page], :, key % page, 0] = 0x7E  # 448
    q = pool.queries(total, heads, dtype)
    clean = q.clone()
    last = news[0] - 1
    bad = [(0, 1, math.nan), (last, heads - 1, math.inf), (total - 1, 0, math.nan)]
    for row, head, x in bad:
        q[row, head, 3] = x
    if dtype == BF16:
        q[last, 2] = 0
        q[last, 2, 0] = 3e38
        bad.append((last, 2, 0))
    got, indptr = pool.attend(q, lens, news)
    want, tol = R.ref_attention_by_head(clean, pool.rows("k", lens), pool.rows("v", lens), lens, indptr, dim ** -0.5, half_step=HALF[dtype],
                                        v_scale=pool.scales(lens))
    spoilt = torch.zeros(total, heads, dtype=torch.bool, device=device)
    for row, head, _ in bad:
        spoilt[row, head] = True
    assert not bool(torch.isfinite(got[spoilt]).any())
    assert bool(((got[~spoilt].double() - want[~spoilt]).abs() <= tol[~spoilt]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("form,dim", CASES)
@pytest.mark.parametrize("page", [16, 32, 64])
def test_lengths_beyond_the_table_see_what_the_table_has(device, form, dim, page):
    """Tables that end inside a step of 64 keys, lengths behind their end."""
    heads, group, _, (lens, news) = FORMS[form]
    width = (max(lens) // page - 1) // 2 * 2 + 1
    capacity = width * page
    assert form_of(sum(news), heads * group, len(lens), heads, dim, page, width)[0] == form[0]
    pool = Forms(device, width * len(lens), heads, page, dim, len(lens), width)
    pool.fill([capacity] + lens[1:], [capacity] + lens[1:])
    q = pool.queries(sum(news), heads * group, BF16)
    for beyond in (1, 40, 64, 1000):
        pool.check(q, [capacity + beyond] + lens[1:], news)
        pool.check(q, [capacity + beyond] + lens[1:], news, window=500, sinks=20)


@pytest.mark.gpu
@pytest.mark.parametrize("form,dim", CASES)
@pytest.mark.parametrize("page,run", [(16, 1), (64, 1), (64, 9)])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("small", [0.003, 0.0])
def test_rows_on_pages_of_very_different_sizes(device, form, dim, page, run, dtype, small):
    """Values of 30000 in every other page (or run of pages, so that a wave that takes every eighth step meets both) and of 0.003 or
    zero between them, scales 2^23 or 2^48 apart: rows whose weight lies on the small ones, beside rows on the large ones and rows on both."""
    heads, group, _, (lens, news) = FORMS[form]
    width = -(-max(lens) // page)
    assert form_of(sum(news), heads * group, len(lens), heads, dim, page, width)[0] == form[0]
    pool = Forms(device, width * len(lens), heads, page, dim, len(lens), width)
    indptr = [0] + list(itertools.accumulate(lens))
    k, v = (torch.randn(indptr[-1], heads, dim, generator=pool.g) for _ in range(2))
    odd = torch.cat([torch.arange(n) // page // run % 2 for n in lens])[:, None]
    k[..., 0] = 8.0 * odd - 4.0
    v = v.clamp(-2, 2) * torch.where(odd == 1, small, 30000.0)[..., None]
    i32 = pool.i32
    ops.kv_cache_append(pool.cache, k.to(dtype).to(device), v.to(dtype).to(device), i32(pool.table), i32(lens), i32(indptr))
    assert float(pool.cache.v_scale[pool.table[0][0], 0] / pool.cache.v_scale[pool.table[0][run], 0]) >= 2.0 ** 22
    q = torch.randn(sum(news), heads * group, dim, generator=pool.g) * 0.1
    q[..., 0] = torch.randint(-1, 2, q.shape[:2], generator=pool.g) * 10.0
    q[0, :, 0] = 10.0
    pool.check(q.to(dtype).to(device), lens, news, sm_scale=1.0)


def _described(ptr, shape, strides, dtype):
    """A descriptor of a tensor that does not exist (for refusals, which look at nothing else)."""
    d = _lib.TgTensor()
    d.ptr, d.ndim, d.dtype = ptr, len(shape), dtype
    for i, (n, s) in enumerate(zip(shape, strides)):
        d.shape[i], d.strides[i] = n, s
    return ctypes.byref(d)


def _rc_of_sizes(tokens, q_heads, kv_heads, dim, batch=1, width=1, page=16):
    """What attention over sizes that no memory holds returns: -4 (there is no device 999) where it would have gone on to launch."""
    dense = lambda *s: (s, [math.prod(s[i + 1:]) for i in range(len(s))])  # noqa: E731
    t = lambda dtype, *s: _described(1 << 20, *dense(*s), dtype)  # noqa: E731
    codes = {d: _lib.make_tensor_desc(torch.zeros(1, dtype=d)).dtype for d in (BF16, torch.float8_e4m3fn, torch.float32, torch.int32)}
    e4m3, f32, i32 = codes[torch.float8_e4m3fn], codes[torch.float32], codes[torch.int32]
    x = t(codes[BF16], tokens, q_heads, dim)
    out = _described(1 << 21, *dense(tokens, q_heads, dim), codes[BF16])
    rc = _lib.load().tg_fp8_kv_attention(out, x, t(e4m3, 1, kv_heads, page, dim), t(e4m3, 1, kv_heads, dim, page), t(f32, 1, kv_heads), t(f32, 1, kv_heads),
                                         t(i32, batch, width), t(i32, batch), t(i32, batch + 1), 1.0, 0, 0, None, 999, 0)
    return rc, _lib.load().tg_last_error().decode()


def test_launches_are_refused_by_the_threads_that_they_have():
    # no join where contexts are whole: 2^34 elements and more of a result are no reason
    for dim in (64, 128, 256):
        assert form_of(1 << 20, 128, 1, 128, dim, 16, 1) == (128, 1)
        assert _rc_of_sizes(1 << 20, 128, 128, dim)[0] == -4
    # 128-row tiles have 256 threads: 2^23 + 2^22 of them can be launched
    for dim in (64, 128, 256):
        assert _rc_of_sizes(3 << 22, 128, 128, dim)[0] == -4
    tokens = (1 << 28) - 129  # (2^21 - 1 tiles for each of 7 heads)
    assert tokens * 7 <= 2 ** 31 - 1 and form_of(tokens, 7, 1, 7, 64, 16, 1) == (128, 1) and _rc_of_sizes(tokens, 7, 7, 64)[0] == -4
    batch = 1 << 15
    assert form_of(batch, 1024, batch, 1024, 128, 16, 1) == (16, 1)
    rc, said = _rc_of_sizes(batch, 1024, 1024, 128, batch=batch)
    assert rc == -6 and "threads" in said and "kv_cache_attention" in said


@pytest.mark.gpu
def test_a_result_of_more_than_2_to_the_34_elements(device):
    """Contexts that are whole need no join, whose launch would be too large."""
    tokens, heads, dim = 1 << 20, 64, 256
    assert tokens * heads * dim >= 2 ** 34 and form_of(tokens, heads, 1, heads, dim, 16, 1) == (128, 1)
    pool = Forms(device, 1, heads, 16, dim, 1, 1)
    pool.fill([16], [16])
    one = pool.queries(1, heads, BF16)
    got = ops.kv_cache_attention(one.expand(tokens, heads, dim), pool.cache, pool.i32(pool.table), pool.i32([tokens]), pool.i32([0, tokens]))
    want = ops.kv_cache_attention(one.expand(150, heads, dim), pool.cache, pool.i32(pool.table), pool.i32([150]), pool.i32([0, 150]))
    assert form_of(150, heads, 1, heads, dim, 16, 1) == (128, 1)
    assert torch.equal(got[:150], want)
    for at in (1 << 15, (1 << 19) - 3, 1 << 19, tokens - 5):
        assert torch.equal(got[at:at + 5], want[20:21].expand(5, heads, dim))


@pytest.mark.gpu
@pytest.mark.parametrize("form,dim", CASES)
@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_scales_that_are_no_powers_of_two(device, form, dim, page, dtype):
    """A cache that something else than kv_cache_append has filled: any scales, some of them zero."""
    pool, group, lens, news, width = _pool_of(device, form, dim, page, dtype)
    assert form_of(sum(news), pool.heads * group, len(lens), pool.heads, dim, page, width)[0] == form[0]
    for t in (pool.cache.k_scale, pool.cache.v_scale):
        t.mul_((torch.rand(t.shape, generator=pool.g) * 3 + 0.3).to(device))
    pool.cache.v_scale[pool.table[0][1]] = 0
    q = pool.queries(sum(news), pool.heads * group, dtype)
    indptr = [0] + list(itertools.accumulate(news))
    got = ops.kv_cache_attention(q, pool.cache, pool.i32(pool.table), pool.i32(lens), pool.i32(indptr))
    scales = [s.clamp(min=2.0 ** -64) for s in pool.scales(lens)]  # (a scale of zero counts as the least)
    want, tol = R.ref_attention_by_head(q, pool.rows("k", lens), pool.rows("v", lens), lens, indptr, dim ** -0.5, half_step=HALF[dtype], v_scale=scales)
    assert bool(((got.double() - want).abs() <= tol + 448 * 2.0 ** -64).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page,longest", [(32, 1000), (64, 1000), (64, 1500)])
def test_a_prompt_among_decoding_sequences(device, dim, page, longest):
    """The 128-row form with tiles of one token's rows: single tokens, drafted ones, nothing new and no tokens at all beside a prompt."""
    g = torch.Generator().manual_seed(dim + page)
    batch, heads, group = 70, 8, 4
    lens = torch.randint(1, 200, (batch,), generator=g).tolist()
    lens[3], lens[11], lens[20], lens[69] = longest, 0, longest - 1, 70
    news = [1] * batch
    news[3], news[11], news[30], news[31], news[69] = 1000, 0, 0, min(5, lens[31]), 70
    width = -(-longest // page)
    assert form_of(sum(news), heads * group, batch, heads, dim, page, width) == (128, 1)
    pool = Forms(device, sum(-(-n // page) for n in lens) + 1, heads, page, dim, batch, 1)
    pages = iter(torch.randperm(pool.cache.k.shape[0], generator=g).tolist())
    pool.table = [[next(pages) if i * page < n else -1 for i in range(width)] for n in lens]
    pool.fill(lens, lens)
    q = pool.queries(sum(news), heads * group, BF16, 2.0)
    pool.check(q, lens, news)
    pool.check(q, lens, news, window=100, sinks=5)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,heads,group,news", [(16, 2, 4, 3), (32, 2, 5, 180), (128, 8, 4, 281)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_many_faint_keys(device, rows, heads, group, news, dtype):
    """One strong key with value zero beside twenty thousand faint ones with value one, each 2^-25.2 of it, in every form."""
    n, dim, strong = 20000, 64, 20.0
    width = -(-n // 64)
    assert form_of(news, heads * group, 1, heads, dim, 64, width)[0] == rows
    cache = ops.alloc_kv_cache(width, heads, dim, 64, device=device)
    k, v = torch.zeros(n, heads, dim, device=device), torch.ones(n, heads, dim, device=device)
    k[..., 0] = 2.5
    k[0, :, 0], v[0] = strong, 0
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    table = torch.arange(width, dtype=torch.int32, device=device)[None]
    ops.kv_cache_append(cache, k.to(dtype), v.to(dtype), table, i32(n), i32(0, n))
    q = torch.zeros(news, heads * group, dim, dtype=dtype, device=device)
    q[..., 0] = 1
    out = ops.kv_cache_attention(q, cache, table, i32(n), i32(0, news), sm_scale=1.0).cpu().double()
    weight = math.exp(2.5 - strong)
    faint = torch.arange(n - news, n, dtype=torch.float64)[:, None, None]
    want = faint * weight / (1 + faint * weight)
    # a weight is rounded to 16 bits, or by half of f16's smallest step, a 128th of 2^-25 against the maximum; the scores' 20 are 2^-23 off, the
    # exponentials and the sum of 20000 fp32 terms a few units of 2^-24 each
    tol = want * (2 * HALF[dtype] + 20 * 2.0 ** -22 + 20000 / 16 * 2.0 ** -24) + (faint * 2.0 ** -32 if dtype == F16 else 0)
    assert bool(((out - want).abs() <= tol).all())
