"""rms_norm_quant and the paged e4m3 cache: refusals and the oracle on the CPU, the kernels against float64 on a GPU.

Tolerances count roundings: half a step of a type is eps / 2 of the value (bf16 2^-8, f16 2^-11, fp32 2^-24, e4m3 2^-4), and
half of e4m3's smallest step is 2^-10 of the scale."""

import itertools
import math

import pytest
import torch

from oracle import decoder_reference as R
from tilegym_amd import _lib, ops

FP8 = torch.float8_e4m3fn
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


# ---------------------------------------------------------------------------- CPU: the oracle, refusals
def test_oracle_page_scale_and_rope():
    for e in (-40, -7, 0, 13, 40):
        assert R.ref_page_scale(448.0 * 2.0 ** e) == 2.0 ** e
        assert R.ref_page_scale(448.0 * 2.0 ** e * (1 + 2.0 ** -20)) == 2.0 ** min(40, e + 1)
    assert R.ref_page_scale(0.0) == 2.0 ** -40 and R.ref_page_scale(math.inf) == 2.0 ** 40
    # a turn keeps lengths and adds angles
    table = ops.rope_table(50, 32, base=100.0, device="cpu")
    x = torch.randn(1, 2, 64, generator=torch.Generator().manual_seed(1))
    for inter in (False, True):
        y = R.ref_rope(x, [17], table, inter)
        torch.testing.assert_close(y.norm(dim=-1), x.double().norm(dim=-1), rtol=1e-6, atol=0)
        assert torch.equal(y[..., 32:], x[..., 32:].double())
        torch.testing.assert_close(R.ref_rope(y, [20], table, inter), R.ref_rope(x, [37], table, inter), rtol=1e-5, atol=1e-5)


def test_rope_table_is_exact_far_out():
    table = ops.rope_table(1 << 20, 16, device="cpu")
    for p in (0, 1, 999_999, (1 << 20) - 1):
        for i in range(8):
            angle = p * 10000.0 ** (-2 * i / 16)
            assert abs(float(table[p, i]) - math.cos(angle)) < 2e-7 and abs(float(table[p, 8 + i]) - math.sin(angle)) < 2e-7
    half = ops.rope_table(64, 16, position_scale=0.5, device="cpu")
    torch.testing.assert_close(half[::2], ops.rope_table(32, 16, device="cpu"))
    freq = torch.linspace(0.1, 1, 8)
    own = ops.rope_table(9, 16, inv_freq=freq, magnitude=2.0, device="cpu")
    torch.testing.assert_close(own[3], 2 * torch.cat([(3 * freq.double()).cos(), (3 * freq.double()).sin()]).float())
    with pytest.raises(ValueError):
        ops.rope_table(9, 16, inv_freq=freq[:7], device="cpu")
    with pytest.raises(ValueError):
        ops.rope_table(9, 15, device="cpu")


def test_operators_have_no_host_path():
    cache = ops.alloc_kv_cache(2, 1, 64, 16, device="cpu")
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    x = torch.zeros(1, 1, 64, dtype=BF16)
    with pytest.raises(RuntimeError):
        ops.rms_norm_quant(torch.zeros(2, 128), torch.ones(128))
    with pytest.raises(RuntimeError):
        ops.kv_cache_append(cache, x, x, i32(0)[None], i32(1), i32(0, 1))
    with pytest.raises(RuntimeError):
        ops.kv_cache_read(cache, i32(0)[None], i32(0, 1), 1)
    with pytest.raises(RuntimeError):
        ops.kv_cache_attention(x, cache, i32(0)[None], i32(1), i32(0, 1))
    with pytest.raises(NotImplementedError):
        ops.alloc_kv_cache(2, 1, 96, 16, device="cpu")
    with pytest.raises(NotImplementedError):
        ops.alloc_kv_cache(2, 1, 64, 48, device="cpu")


def _norm_rc(x=None, weight=None, q=None, scales=None, scale=None, residual=None, residual_out=None, norm_out=None, eps=1e-6, group=128):
    x = torch.zeros(4, 256, dtype=BF16) if x is None else x
    weight = torch.ones(256, dtype=BF16) if weight is None else weight
    q = torch.zeros(x.shape, dtype=torch.uint8).view(FP8) if q is None else q
    if scales is None and scale is None:
        scales = torch.zeros(4, 2)
    d = _lib._desc
    return _lib.load().tg_fp8_rms_norm_quant(d(q), d(scales), d(norm_out), d(residual_out), d(x), d(weight), d(residual), d(scale), eps, group, 0, 0)


def test_norm_refusals_need_no_device():
    x = torch.zeros(4, 256, dtype=BF16)
    assert _norm_rc(x=x.double().to(torch.int32)) == -2
    assert _norm_rc(weight=torch.ones(256, dtype=F16)) == -2
    assert _norm_rc(weight=torch.ones(128, dtype=BF16)) == -6
    assert _norm_rc(q=torch.zeros(4, 256, dtype=torch.int8)) == -2
    assert _norm_rc(q=torch.zeros(4, 128, dtype=torch.uint8).view(FP8)) == -6
    assert _norm_rc(scales=torch.zeros(4, 3)) == -6
    assert _norm_rc(group=24) == -6
    assert _norm_rc(scale=torch.ones(2)) == -6
    assert _norm_rc(scale=torch.ones(1), scales=torch.zeros(4, 2)) == -6
    assert _norm_rc(scale=torch.ones(1, dtype=F16)) == -2
    assert _norm_rc(residual_out=x) == -6                                  # without residual
    assert _norm_rc(residual=torch.zeros(3, 256, dtype=BF16)) == -6
    assert _norm_rc(residual=torch.zeros(4, 256)) == -2
    assert _norm_rc(eps=-1.0) == -6 and _norm_rc(eps=math.nan) == -6
    assert _norm_rc(x=torch.zeros(4, 512, dtype=BF16)[:, ::2]) == -6       # not contiguous
    assert _norm_rc(x=torch.zeros(4 * 256 + 1, dtype=BF16)[1:].view(4, 256)) == -6  # not aligned
    assert _norm_rc(x=torch.zeros(1, 32768 + 128, dtype=BF16), weight=torch.ones(32768 + 128, dtype=BF16), scales=torch.zeros(1, 257)) == -6
    assert _norm_rc(x=torch.zeros(4, 0, dtype=BF16), weight=torch.ones(0, dtype=BF16), scales=torch.zeros(4, 0)) == -6
    assert _norm_rc(x=torch.zeros(0, 256, dtype=BF16), scales=torch.zeros(0, 2)) == 0


def _cache_args(pages=3, heads=2, page=16, dim=64, batch=2, width=2, tokens=3, q_heads=4, dtype=BF16):
    c = ops.alloc_kv_cache(pages, heads, dim, page, device="cpu") if page in (16, 32, 64, 128) and dim in (64, 128, 256) else ops.KVCache(
        torch.zeros(pages, heads, page, dim, dtype=torch.uint8).view(FP8), torch.zeros(pages, heads, dim, page, dtype=torch.uint8).view(FP8),
        torch.ones(pages, heads), torch.ones(pages, heads))
    return {"k_cache": c.k, "v_cache": c.v, "k_scale": c.k_scale, "v_scale": c.v_scale, "k": torch.zeros(tokens, heads, dim, dtype=dtype),
            "v": torch.zeros(tokens, heads, dim, dtype=dtype), "table": torch.zeros(batch, width, dtype=torch.int32),
            "lens": torch.zeros(batch, dtype=torch.int32), "indptr": torch.zeros(batch + 1, dtype=torch.int32),
            "q": torch.zeros(tokens, q_heads, dim, dtype=dtype), "out": torch.zeros(tokens, q_heads, dim, dtype=dtype),
            "rope": torch.zeros(width * page, dim)}


def _append_rc(a, interleaved=0):
    d = _lib._desc
    return _lib.load().tg_fp8_kv_append(*[d(a[n]) for n in ("k_cache", "v_cache", "k_scale", "v_scale", "k", "v", "table", "lens", "indptr", "out", "q", "rope")],
                                        interleaved, 0, 0)


def _read_rc(a):
    d = _lib._desc
    return _lib.load().tg_fp8_kv_read(*[d(a[n]) for n in ("k", "v", "k_cache", "v_cache", "k_scale", "v_scale", "table", "indptr")], 0, 0)


def _attention_rc(a, scale=1.0, window=0, sinks=0, ws=None):
    d = _lib._desc
    return _lib.load().tg_fp8_kv_attention(*[d(a[n]) for n in ("out", "q", "k_cache", "v_cache", "k_scale", "v_scale", "table", "lens", "indptr")], scale,
                                           window, sinks, d(ws), 0, 0)


def _wrong():
    """(what, changed arguments, code) that every call over the cache refuses."""
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8)  # noqa: E731
    yield "page size", _cache_args(page=48), -6
    yield "head dim", _cache_args(dim=96), -6
    for name, value, rc in (("k_cache", u8(3, 2, 16, 64), -2), ("v_cache", u8(3, 2, 16, 64).view(FP8), -6), ("k_scale", torch.ones(3, 3), -6),
                            ("v_scale", torch.ones(3, 2, dtype=F16), -2), ("table", torch.zeros(2, 2, dtype=torch.int64), -2),
                            ("table", torch.zeros(2, 0, dtype=torch.int32), -6), ("table", torch.zeros(2, 4, dtype=torch.int32)[:, ::2], -6),
                            ("indptr", torch.zeros(2, dtype=torch.int32), -6), ("indptr", torch.zeros(3, dtype=torch.int64), -2), ("k_cache", None, -5),
                            ("k_cache", u8(6, 2, 16, 64).view(FP8)[::2], -6)):
        yield name, {**_cache_args(), name: value}, rc
    yield "no pages", _cache_args(pages=0), -6


def test_cache_refusals_need_no_device():
    for what, args, rc in _wrong():
        for call in (_append_rc, _read_rc, _attention_rc):
            assert call(args) == rc, (what, call.__name__)
    a = _cache_args()
    with_ = lambda **kw: {**a, **kw}  # noqa: E731
    for call in (_append_rc, _attention_rc):
        assert call(with_(lens=torch.zeros(3, dtype=torch.int32))) == -6
        assert call(with_(lens=None)) == -5
    # k and v
    assert _append_rc(with_(k=a["k"].float())) == -2 and _append_rc(with_(v=a["v"].to(F16))) == -2
    assert _append_rc(with_(k=torch.zeros(3, 1, 64, dtype=BF16))) == -6 and _append_rc(with_(v=torch.zeros(2, 2, 64, dtype=BF16))) == -6
    assert _append_rc(with_(k=torch.zeros(3, 2, 128, dtype=BF16)[..., ::2])) == -6
    assert _append_rc(with_(k=torch.zeros(3, 2, 68, dtype=BF16)[..., :64])) == -6             # heads off 16-byte boundaries
    assert _append_rc(with_(k=torch.zeros(3 * 2 * 64 + 1, dtype=BF16)[1:].view(3, 2, 64))) == -6
    # rope and q
    assert _append_rc(with_(rope=None)) == -5                                                 # q without it
    assert _append_rc(with_(rope=None, q=None)) == -5 and _append_rc(with_(out=None)) == -5
    for rope in (torch.zeros(31, 64), torch.zeros(32, 24), torch.zeros(32, 80), torch.zeros(32, 0)):
        assert _append_rc(with_(rope=rope)) == -6
    assert _append_rc(with_(rope=torch.zeros(32, 64, dtype=F16))) == -2
    assert _append_rc(with_(out=a["q"])) == -6                                                # in place
    assert _append_rc(with_(q=a["q"].to(F16), out=a["out"].to(F16))) == -2
    assert _append_rc(with_(out=torch.zeros(3, 5, 64, dtype=BF16))) == -6
    # reading
    assert _read_rc(with_(k=torch.zeros(3, 2, 64, dtype=torch.int32))) == -2 and _read_rc(with_(v=a["v"].float())) == -2
    assert _read_rc(with_(v=torch.zeros(4, 2, 64, dtype=BF16))) == -6
    # attention
    assert _attention_rc(with_(q=a["q"].float(), out=a["out"].float())) == -2 and _attention_rc(with_(out=a["out"].to(F16))) == -2
    assert _attention_rc(with_(q=torch.zeros(3, 3, 64, dtype=BF16), out=torch.zeros(3, 3, 64, dtype=BF16))) == -6  # heads
    assert _attention_rc(with_(out=a["q"])) == -6
    assert _attention_rc(a, scale=math.inf) == -6 and _attention_rc(a, scale=math.nan) == -6
    assert _attention_rc(a, window=-1) == -6 and _attention_rc(a, window=4, sinks=-1) == -6 and _attention_rc(a, sinks=4) == -6
    # a long table: splits, and so a workspace
    long = _cache_args(width=1000)
    need = _lib.load().tg_fp8_kv_attention_workspace_bytes(3, 4, 2, 2, 64, 16, 1000, 0, 0)
    assert need > 0 and need % 4 == 0
    assert _attention_rc(long) == -5 and _attention_rc(long, ws=torch.zeros(need - 1, dtype=torch.uint8)) == -6
    assert _lib.load().tg_fp8_kv_attention_workspace_bytes(3, 4, 2, 2, 64, 16, 2, 0, 0) == 0
    assert _lib.load().tg_fp8_kv_attention_workspace_bytes(3, 5, 2, 2, 64, 16, 2, 0, 0) == 0
    # nothing to do, no device needed
    assert _append_rc(_cache_args(tokens=0)) == 0 and _read_rc(_cache_args(tokens=0)) == 0 and _attention_rc(_cache_args(tokens=0)) == 0
    assert _append_rc(_cache_args(batch=0)) == 0 and _read_rc(_cache_args(batch=0)) == 0 and _attention_rc(_cache_args(batch=0)) == 0


# ---------------------------------------------------------------------------- norm
NORM_SHAPES = [(1, 16), (1, 128), (5, 512), (3, 1024), (7, 1040), (4, 2048), (9, 4096), (2, 5120), (3, 8192), (2, 8208), (3, 16384), (2, 32768), (1000, 256)]


def _norm_case(rows, hidden, dtype, device, seed=0):
    g = torch.Generator().manual_seed(seed + rows * hidden)
    x = torch.randn(rows, hidden, generator=g)
    x = torch.where(torch.rand(rows, hidden, generator=g) < 0.01, x * 30, x).to(dtype)
    r = (torch.randn(rows, hidden, generator=g) * 3).to(dtype)
    w = (1 + 0.3 * torch.randn(hidden, generator=g)).to(dtype)
    return x.to(device), r.to(device), w.to(device)


def _check_norm(out, x, w, eps, residual, group, scale, dtype, norm=False):
    out = [t.cpu() for t in out]
    x, w, residual = x.cpu(), w.cpu(), None if residual is None else residual.cpu()
    s, y = R.ref_rms_norm(x, w, eps, residual)
    q, scales = out[0].double(), out[1].double()
    # at most 64 squares in a row per lane, 6 + 8 sums over lanes and waves, the mean, root, reciprocal and two products: 46 halves of 2^-23
    rel = 2.0 ** -18
    if scale is None:
        want = R.ref_group_scales(y, group)
        assert bool(((scales - want).abs() <= rel * want).all())
        scales = scales.repeat_interleave(group, -1)
    step = scales * 2.0 ** -10
    limit = y.clamp(-448 * scales, 448 * scales) if scale is not None else y
    assert bool(((q * scales - limit).abs() <= (2.0 ** -4 + 2 * rel) * limit.abs() + step).all())
    rest = out[2:]
    if residual is not None:
        assert bool(((rest[0].double() - s).abs() <= HALF[dtype] * (1 + 2.0 ** -10) * s.abs() + 2.0 ** -24 * s.abs() + 2.0 ** -26).all())
        rest = rest[1:]
    if norm:
        assert bool(((rest[0].double() - y).abs() <= (HALF[dtype] + rel) * y.abs() + 2.0 ** -26).all())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,hidden", NORM_SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_norm(device, rows, hidden, dtype):
    x, r, w = _norm_case(rows, hidden, dtype, device)
    for group in (16, 32, 64, 128):
        if hidden % group:
            continue
        _check_norm(ops.rms_norm_quant(x, w, 1e-5, group_size=group), x, w, 1e-5, None, group, None, dtype)
        _check_norm(ops.rms_norm_quant(x, w, 1e-5, residual=r, group_size=group, return_norm=True), x, w, 1e-5, r, group, None, dtype, True)
    scale = torch.tensor([0.02], device=device)
    out = ops.rms_norm_quant(x, w, 1e-5, residual=r, group_size=None, scale=scale)
    assert out[1] is scale
    _check_norm(out, x, w, 1e-5, r, None, scale, dtype)
    if dtype != F32:
        _check_norm(ops.rms_norm_quant(x, w.float(), 1e-5, residual=r, group_size=16), x, w.float(), 1e-5, r, 16, None, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_norm_in_place_and_odd_values(device, dtype):
    x, r, w = _norm_case(6, 1024, dtype, device)
    x[2], r[2] = 0, 0                       # a row of zeros: scales 1, codes 0
    x[3, 128:256], r[3, 128:256] = 0, 0     # a group of zeros
    want = ops.rms_norm_quant(x, w, 1e-6, residual=r)
    assert bool((want[0][2].float() == 0).all()) and bool((want[1][2] == 1).all()) and float(want[1][3, 1]) == 1
    for target in ("x", "residual"):
        x2, r2 = x.clone(), r.clone()
        got = ops.rms_norm_quant(x2, w, 1e-6, residual=r2, residual_out=x2 if target == "x" else r2)
        assert got[2] is (x2 if target == "x" else r2)
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))
    # a leading shape of its own, no rows, and what is refused
    got = ops.rms_norm_quant(x.view(2, 3, 1024), w, 1e-6, residual=r.view(2, 3, 1024))
    assert got[0].shape == (2, 3, 1024) and got[1].shape == (2, 3, 8) and torch.equal(got[1].view(6, 8), want[1])
    empty = ops.rms_norm_quant(x[:0], w, 1e-6)
    assert empty[0].shape == (0, 1024) and empty[1].shape == (0, 8)
    # an infinite element spoils its own row only
    x[4, 5] = math.inf
    got = ops.rms_norm_quant(x, w, 1e-6, residual=r)
    keep = [0, 1, 2, 3, 5]
    assert torch.equal(got[0].view(torch.uint8)[keep], want[0].view(torch.uint8)[keep]) and torch.equal(got[1][keep], want[1][keep])
    with pytest.raises(_lib.TileGymHipError):
        ops.rms_norm_quant(x[:, ::2], w[::2].contiguous())
    with pytest.raises(ValueError):
        ops.rms_norm_quant(x, w, residual_out=r)
    with pytest.raises(ValueError):
        ops.rms_norm_quant(x, w.cpu())
    with pytest.raises(NotImplementedError):
        ops.rms_norm_quant(x, w, group_size=48)


# ---------------------------------------------------------------------------- cache
class Pool:
    """A cache on the device beside the oracle's, its unwritten slots full of NaN codes and its unwritten scales NaN."""

    def __init__(self, device, pages, heads, page, dim, batch, width, seed=0):
        self.cache = ops.alloc_kv_cache(pages, heads, dim, page, device=device)
        for t in self.cache[:2]:
            t.view(torch.uint8).fill_(0x7F)
        for t in self.cache[2:]:
            t.fill_(math.nan)
        self.ref = R.RefCache(pages, heads, page, dim)
        self.device, self.heads, self.page, self.dim = device, heads, page, dim
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
        self.table = [[order.pop() if order else -1 for _ in range(width)] for _ in range(batch)]
        self.g = torch.Generator().manual_seed(seed + 1)

    def i32(self, v):
        return torch.tensor(v, dtype=torch.int32, device=self.device)

    def fill(self, lens, news, dtype=BF16, rope=None, interleaved=False, q_heads=None, spread=True, pad=0):
        """Append `news` tokens so that sequences have `lens`; returns (q in, q out)."""
        indptr = [0] + list(itertools.accumulate(news))
        total, heads = indptr[-1] + pad, self.heads
        qh = q_heads or heads
        qkv = torch.randn(total, qh + 2 * heads, self.dim, generator=self.g)
        if spread:  # tokens and heads of different sizes: scales move
            qkv = qkv * 2.0 ** torch.randint(-3, 4, (total, qh + 2 * heads, 1), generator=self.g)
        qkv = qkv.to(dtype)
        dev = qkv.to(self.device)
        q, k, v = dev[:, :qh], dev[:, qh:qh + heads], dev[:, qh + heads:]
        out = ops.kv_cache_append(self.cache, k, v, self.i32(self.table), self.i32(lens), self.i32(indptr), q=q if rope is not None else None,
                                  rope=None if rope is None else rope.to(self.device), interleaved=interleaved)
        kr, qr = qkv[:, qh:qh + heads].double(), qkv[:, :qh].double()
        if rope is not None:
            pos = [p for n, length in zip(news, lens) for p in range(length - n, length)] + [0] * pad
            kr, qr = R.ref_rope(kr, pos, rope, interleaved), R.ref_rope(qr, pos, rope, interleaved)
        self.ref.append(kr, qkv[:, qh + heads:], self.table, lens, indptr)
        return q, out, qr, indptr

    def check(self, turned):
        """Scales exactly, elements within one rounding (turned: and fp32's three), unwritten slots untouched."""
        for name, codes, scales in (("k", self.cache.k, self.cache.k_scale), ("v", self.cache.v.transpose(-1, -2), self.cache.v_scale)):
            want, unit = self.ref.value[name], self.ref.scale[name]
            written = ~torch.isnan(want)
            pages = written.flatten(2).any(-1)
            assert torch.equal(scales.cpu().double()[pages], unit[pages])
            got = codes.cpu().float().double() * scales.cpu().double()[..., None, None]
            raw = codes.contiguous().view(torch.uint8).cpu()
            assert bool((raw[~written] == 0x7F).all())
            assert not bool((raw[written] == 0x7F).any())
            x = want[written]
            top = (448 * unit[..., None, None]).expand_as(want)[written]
            step = (unit[..., None, None] * 2.0 ** -10).expand_as(want)[written]
            x = torch.minimum(torch.maximum(x, -top), top)
            # a turned element is a difference of two products: off by 2^-22 of its page's largest
            slack = 2.0 ** -22 * top * math.sqrt(2) if turned and name == "k" else 0 * top
            assert bool(((got[written] - x).abs() <= 2.0 ** -4 * x.abs() * (1 + 2.0 ** -10) + 2 * step + slack).all())

    def rows(self, name, lens):
        """What the device's cache holds, per sequence (positions, heads, D) in float64; zeros in pages that are not there."""
        codes, scales = (self.cache.k, self.cache.k_scale) if name == "k" else (self.cache.v.transpose(-1, -2), self.cache.v_scale)
        x = (codes.float().double() * scales.double()[..., None, None]).cpu()
        out = []
        for b, n in enumerate(lens):
            parts = [x[p].transpose(0, 1) if 0 <= p < x.shape[0] else torch.full((self.page, self.heads, self.dim), math.nan, dtype=torch.float64)
                     for p in self.table[b]]
            out.append(torch.cat(parts)[:n])
        return out


CACHES = [(16, 64, 1), (16, 128, 2), (32, 128, 3), (64, 64, 2), (64, 128, 8), (64, 256, 1), (128, 128, 2), (128, 256, 2)]


@pytest.mark.gpu
@pytest.mark.parametrize("page,dim,heads", CACHES)
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rotary", [None, "half", "pairs", "part"])
def test_append(device, page, dim, heads, dtype, rotary):
    batch, width = 5, 4
    pool = Pool(device, 22, heads, page, dim, batch, width, seed=page + dim + heads)
    rope = None
    if rotary:
        r = 32 if rotary == "part" else dim
        rope = ops.rope_table(width * page, r, base=500.0, device="cpu")
    inter = rotary in ("pairs", "part")
    # a first chunk (none, one token, a page, a page and one, most of the table), single tokens, another chunk over page borders
    lens = [0, 1, page, page + 1, 3 * page - 2]
    for step, news in enumerate([lens, [1] * 5, [1, 0, 1, 0, 1], [page, 3, 2 * page - 3, 17, 5], [1, 1, 0, 1, 1]]):
        if step:
            lens = [a + b for a, b in zip(lens, news)]
        q, out, want, indptr = pool.fill(lens, news, dtype, rope, inter, q_heads=heads * 3 + 1)
        pool.check(rotary is not None)
        if rope is None:
            assert out is None
        elif indptr[-1]:
            got = out.cpu().double()
            slack = 2.0 ** -22 * 2 * want.abs().amax()  # two products and a difference in fp32
            assert out.shape == q.shape and bool(((got - want).abs() <= HALF[dtype] * want.abs() * (1 + 2.0 ** -10) + slack + 2.0 ** -26).all())


@pytest.mark.gpu
def test_append_values_at_the_edges(device):
    """Zeros, infinities, NaN, magnitudes at a power of two's border, and beyond the scales' range."""
    pool = Pool(device, 8, 1, 16, 64, 7, 1)
    x = torch.zeros(7, 1, 64)
    x[1, 0, 3] = 448.0                 # exactly 448 * 2^0
    x[2, 0, 3] = 450.0                 # one bf16 step above
    x[3, 0, 3] = math.inf
    x[3, 0, 4] = 5.0
    x[4, 0, 3], x[4, 0, 5] = math.nan, 3.5
    x[5, 0, 3] = 3e38
    x[6, 0, 3] = 1e-30
    kv = x.to(BF16).to(device)
    ops.kv_cache_append(pool.cache, kv, kv, pool.i32(pool.table), pool.i32([1] * 7), pool.i32(list(range(8))))
    at = [row[0] for row in pool.table]
    for codes, scale in ((pool.cache.k, pool.cache.k_scale), (pool.cache.v.transpose(-1, -2), pool.cache.v_scale)):
        s, c = scale.cpu()[at, 0].double(), codes.cpu().float()[at, 0, 0]
        assert s.tolist() == [2.0 ** -40, 1.0, 2.0, 2.0 ** 40, 2.0 ** -7, 2.0 ** 40, 2.0 ** -40]
        assert not bool(torch.isnan(c).any()) and bool((c[0] == 0).all())
        assert c[1, 3] == 448 and c[2, 3] == 224 and c[3, 3] == 448 and c[4, 3] == -448 and c[4, 5] == 448 and c[5, 3] == 448 and c[6, 3] == 0


@pytest.mark.gpu
def test_append_leaves_out_what_is_out_of_range(device):
    """Table entries outside the pool, lengths beyond the table, more new tokens than the sequence has, rows of no sequence."""
    pool = Pool(device, 6, 2, 16, 64, 4, 2)
    pool.table = [[0, -1], [1, 99], [2, 3], [4, 5]]
    rope = ops.rope_table(32, 64, device="cpu")
    news, lens = [20, 20, 5, 40], [20, 20, 2, 40]
    indptr = [3] + [3 + n for n in itertools.accumulate(news)]
    g = torch.Generator().manual_seed(0)
    k, v, q = (torch.randn(indptr[-1] + 4, h, 64, generator=g).to(BF16) for h in (2, 2, 3))
    ops.kv_cache_append(pool.cache, k.to(device), v.to(device), pool.i32(pool.table), pool.i32(lens), pool.i32(indptr), q=q.to(device),
                        rope=rope.to(device))
    ref_k = k.double()
    for b, n in enumerate(news):
        for t in range(n):
            p = lens[b] - n + t
            if 0 <= p < 32:
                ref_k[indptr[b] + t] = R.ref_rope(k[indptr[b] + t][None], [p], rope, False)[0]
    pool.ref.append(ref_k, v, pool.table, [min(n, 32) if i != 3 else 40 for i, n in enumerate(lens)], indptr)
    pool.check(True)
    # an indptr that is no prefix sum stays inside the tensors
    for bad in ([0, 70, 30, 9, 20], [-5, 3, 1000, 2000, 3000], [50, 40, 30, 20, 10]):
        ops.kv_cache_append(pool.cache, k.to(device), v.to(device), pool.i32(pool.table), pool.i32([5, -3, 2 ** 31 - 1, 7]), pool.i32(bad),
                            q=q.to(device), rope=rope.to(device))
        torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("page,dim,heads", CACHES)
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_read(device, page, dim, heads, dtype):
    pool = Pool(device, 20, heads, page, dim, 5, 4)
    lens = [1, 2 * page, 3 * page - 5, 0, page + 9]
    pool.fill(lens, lens)
    count = [1, 2 * page, page + 1, 0, page]
    indptr = [0] + list(itertools.accumulate(count))
    k_out, v_out = (torch.full((indptr[-1] + 3, heads, dim), 7.0, dtype=dtype, device=device) for _ in range(2))
    k, v = ops.kv_cache_read(pool.cache, pool.i32(pool.table), pool.i32(indptr), indptr[-1] + 3, dtype, k_out, v_out)
    assert k is k_out and v is v_out
    for name, got in (("k", k), ("v", v)):
        want = torch.cat([x[:n] for x, n in zip(pool.rows(name, lens), count)])
        assert torch.equal(got[:-3].cpu(), want.to(dtype)) and bool((got[-3:] == 7).all())  # one rounding; rows of no sequence untouched
    again = ops.kv_cache_read(pool.cache, pool.i32(pool.table), pool.i32(indptr), indptr[-1], dtype)
    assert torch.equal(again[0], k[:-3]) and torch.equal(again[1], v[:-3])
    with pytest.raises(ValueError):
        ops.kv_cache_read(pool.cache, pool.i32(pool.table), pool.i32(indptr), indptr[-1], dtype, k_out)
    # pages that are not there: their rows are left as they were; an indptr that is no prefix sum stays inside
    table = [row[:] for row in pool.table]
    table[1][0], table[1][1] = -1, 20
    k_out.fill_(7.0), v_out.fill_(7.0)
    ops.kv_cache_read(pool.cache, pool.i32(table), pool.i32(indptr), indptr[-1] + 3, dtype, k_out, v_out)
    assert bool((k_out[1:1 + 2 * page] == 7).all()) and bool((v_out[1:1 + 2 * page] == 7).all()) and torch.equal(k_out[1 + 2 * page:-3], again[0][1 + 2 * page:])
    for bad in ([9, -4, 5000, 3, 0, 7], [0, 4000, 4000, 4000, 4000, 4000]):
        ops.kv_cache_read(pool.cache, pool.i32(pool.table), pool.i32(bad), indptr[-1] + 3, dtype, k_out, v_out)
        torch.cuda.synchronize()


# ---------------------------------------------------------------------------- attention
def _attend(pool, lens, news, group, dtype, window=0, sinks=0, sm_scale=None, q_scale=1.0, out=None, table=None):
    indptr = [0] + list(itertools.accumulate(news))
    heads = pool.heads * group
    wide = torch.randn(indptr[-1], heads + 3, pool.dim, generator=pool.g) * q_scale
    q = wide.to(dtype).to(pool.device)[:, 2:2 + heads]
    got = ops.kv_cache_attention(q, pool.cache, pool.i32(table or pool.table), pool.i32(lens), pool.i32(indptr), sm_scale=sm_scale, window=window,
                                 sink_tokens=sinks, out=out)
    scale = pool.dim ** -0.5 if sm_scale is None else sm_scale
    unit = float(pool.cache.v_scale[~torch.isnan(pool.cache.v_scale)].max()) if bool((~torch.isnan(pool.cache.v_scale)).any()) else 0.0
    want, tol = R.ref_attention(q.cpu(), pool.rows("k", lens), pool.rows("v", lens), lens, indptr, scale, window, sinks, HALF[dtype], unit)
    err = (got.cpu().double()[:indptr[-1]] - want).abs()
    assert bool((err <= tol).all()), (float((err / tol).max()), lens, news)
    return q, got, indptr


LENGTHS = [
    # (lengths, new tokens): decoding from the first token on; a page's and a step's borders
    ([1, 2, 15, 16, 17, 63, 64, 65], [1] * 8),
    # verification of a few tokens, sequences without new ones, a whole short prompt
    ([300, 129, 40, 7, 513], [3, 0, 5, 7, 2]),
    # chunks over a step's border, a prompt from its first token
    ([70, 200, 1], [70, 33, 1]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("page,dim,heads", CACHES)
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lens,news", LENGTHS)
def test_attention(device, page, dim, heads, dtype, lens, news):
    width = -(-max(lens) // page) + 1
    pool = Pool(device, width * len(lens) + 3, heads, page, dim, len(lens), width, seed=dim)
    pool.fill(lens, lens, dtype)
    group = {1: 5, 2: 4, 3: 1, 8: 2}[heads]
    _attend(pool, lens, news, group, dtype)
    _attend(pool, lens, news, group, dtype, window=20, sinks=3)


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 5), (16, 16), (50, 0), (63, 64), (64, 1), (65, 200), (100, 130), (4000, 4)])
@pytest.mark.parametrize("page,group", [(16, 16), (64, 3)])
def test_attention_window(device, window, sinks, page, group):
    lens, news = [700, 64, 129, 333, 1], [1, 9, 40, 2, 1]
    width = -(-max(lens) // page)
    pool = Pool(device, width * 5, 2, page, 64, 5, width)
    pool.fill(lens, lens)
    # pages that no new token sees are not there
    table = [row[:] for row in pool.table]
    for b, (length, n) in enumerate(zip(lens, news)):
        for i in range(width):
            seen = any(j <= p and (p - j < window or j < sinks) for p in range(length - n, length) for j in range(i * page, min((i + 1) * page, length)))
            if not seen:
                table[b][i] = -1 if i % 2 else 10 ** 6
    _attend(pool, lens, news, group, BF16, window, sinks, table=table)


@pytest.mark.gpu
@pytest.mark.parametrize("group,heads,dim", [(1, 1, 128), (7, 2, 64), (16, 1, 128), (17, 1, 64), (32, 1, 128), (48, 1, 64), (4, 8, 128)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attention_long(device, group, heads, dim, dtype):
    """Contexts that are split over workgroups and joined; a table much wider than the lengths; large and tiny scores."""
    lens, news = [2100, 5, 0, 1500], [1, 2, 0, 6]
    pool = Pool(device, 200, heads, 32, dim, 4, 300)
    lens_written = [2100, 5, 0, 1500]
    pool.table = [row[:66] + [-1] * 234 for row in pool.table[:1]] + [[150] + [-1] * 299, [-1] * 300, list(range(151, 198)) + [-1] * 253]
    free = [p for p in range(150)]
    pool.table[0] = free[:66] + [-1] * 234
    pool.fill(lens_written, lens_written, dtype)
    _attend(pool, lens, news, group, dtype)
    _attend(pool, lens, news, group, dtype, q_scale=20.0)
    _attend(pool, lens, news, group, dtype, sm_scale=0.0)
    _attend(pool, lens, news, group, dtype, sm_scale=-0.3)
    _attend(pool, lens, news, group, dtype, window=700, sinks=4)


@pytest.mark.gpu
def test_attention_many_rows(device):
    """A prompt's rows over a context: more than one tile of rows of every form."""
    for page, dim, heads, group, lens, news in [(64, 128, 2, 4, [400, 330], [260, 130]), (16, 64, 1, 8, [190, 20], [150, 20]), (128, 256, 1, 3, [300], [290])]:
        for dtype, window, sinks in [(BF16, 0, 0), (F16, 0, 0), (BF16, 100, 7)]:
            width = -(-max(lens) // page)
            pool = Pool(device, width * len(lens), heads, page, dim, len(lens), width)
            pool.fill(lens, lens, dtype)
            _attend(pool, lens, news, group, dtype, window, sinks)


@pytest.mark.gpu
def test_attention_rows_that_see_nothing_and_rows_of_no_sequence(device):
    pool = Pool(device, 12, 2, 16, 64, 3, 4)
    pool.fill([20, 40, 33], [20, 40, 33])
    # sequence 0 says it has fewer tokens than are new; sequence 1's first page is not there; lengths beyond the table are cut
    table = [row[:] for row in pool.table]
    table[1][0] = -1
    lens, news = [2, 17, 33], [5, 3, 1]
    indptr = [2, 7, 10, 11]
    q = torch.randn(15, 4, 64, generator=pool.g).to(BF16).to(device)
    out = torch.full((15, 4, 64), 3.0, dtype=BF16, device=device)
    got = ops.kv_cache_attention(q, pool.cache, pool.i32(table), pool.i32(lens), pool.i32(indptr), out=out)
    assert got is out
    assert bool((out[:2] == 3).all()) and bool((out[11:] == 3).all())
    assert bool((out[2:5] == 0).all())                        # positions -3 .. -1
    assert bool((out[7:9] == 0).all())                        # positions 14, 15: only the page that is not there
    k, v = pool.rows("k", [2, 40, 33]), pool.rows("v", [2, 40, 33])
    k[1], v[1] = k[1][16:17], v[1][16:17]
    for rows, b, length in ((slice(5, 7), 0, 2), (slice(9, 10), 1, 1), (slice(10, 11), 2, 33)):
        n = rows.stop - rows.start
        want, tol = R.ref_attention(q[rows].cpu(), [k[b]], [v[b]], [length], [0, n], 0.125, half_step=2.0 ** -8)
        assert bool(((out[rows].cpu().double() - want).abs() <= tol).all())
    # nothing at all is there
    empty = ops.kv_cache_attention(q, pool.cache, pool.i32([[-1] * 4] * 3), pool.i32(lens), pool.i32(indptr))
    assert bool((empty[2:11] == 0).all())
    # tensors that contradict each other stay inside their memory
    for bad_ptr, bad_len in (([9, 3, 200, 1], [5, -7, 2 ** 31 - 1]), ([0, 15, 15, 15], [2 ** 31 - 1] * 3), ([-9, 20, 30, 40], [40, 40, 40])):
        ops.kv_cache_attention(q, pool.cache, pool.i32(table), pool.i32(bad_len), pool.i32(bad_ptr))
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_attention_does_not_depend_on_unwritten_slots_or_on_the_call(device):
    """The same bits with other garbage, from another stream, and call after call."""
    lens, news = [333, 70, 1200], [4, 70, 1]
    pool = Pool(device, 60, 2, 32, 128, 3, 40)
    pool.table = [list(range(11)) + [-1] * 29, list(range(11, 14)) + [-1] * 37, list(range(14, 52)) + [-1] * 2]
    pool.fill(lens, lens)
    q, first, indptr = _attend(pool, lens, news, 4, BF16)
    for c, ref in ((pool.cache.k, pool.ref.value["k"]), (pool.cache.v, pool.ref.value["v"].transpose(-1, -2))):
        c.view(torch.uint8)[torch.isnan(ref).to(device)] = 0x35
    args = (pool.cache, pool.i32(pool.table), pool.i32(lens), pool.i32(indptr))
    assert torch.equal(ops.kv_cache_attention(q, *args), first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = ops.kv_cache_attention(q, *args)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again, first)


@pytest.mark.gpu
def test_offsets_beyond_32_bits(device):
    """A pool of more than 4 GiB per half: the last pages are written, read and attended to like the first."""
    pages, heads, page, dim = 70_000, 8, 64, 128
    assert pages * heads * page * dim > 2 ** 32
    cache = ops.KVCache(*(torch.empty(s, dtype=torch.uint8, device=device).view(FP8) for s in ((pages, heads, page, dim), (pages, heads, dim, page))),
                        *(torch.ones(pages, heads, device=device) for _ in range(2)))
    small = Pool(device, 4, heads, page, dim, 1, 3)
    small.table = [[2, 0, 3]]
    far = [[pages - 1, 3, pages - 7]]
    lens, indptr = [150], [0, 150]
    k, v = (torch.randn(150, heads, dim, generator=small.g).to(BF16).to(device) for _ in range(2))
    q = torch.randn(2, 32, dim, generator=small.g).to(BF16).to(device)
    got = []
    for c, table in ((small.cache, small.table), (cache, far)):
        ops.kv_cache_append(c, k, v, small.i32(table), small.i32(lens), small.i32(indptr))
        got.append(ops.kv_cache_read(c, small.i32(table), small.i32(indptr), 150) + (ops.kv_cache_attention(q, c, small.i32(table), small.i32(lens), small.i32([0, 2])),))
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.gpu
def test_many_sequences(device):
    """More sequences than one ballot covers, most of them without new tokens."""
    batch, page = 300, 16
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 40, (batch,), generator=g).tolist()
    pool = Pool(device, batch * 3, 1, page, 64, batch, 3)
    pool.fill(lens, lens)
    pool.check(False)
    news = [min(n, int(torch.randint(0, 3, (1,), generator=g))) if b % 3 else 0 for b, n in enumerate(lens)]
    _attend(pool, lens, news, 4, BF16)
    indptr = [0] + list(itertools.accumulate(lens))
    k, v = ops.kv_cache_read(pool.cache, pool.i32(pool.table), pool.i32(indptr), indptr[-1], F32)
    assert torch.equal(k.cpu().double(), torch.cat(pool.rows("k", lens))) and torch.equal(v.cpu().double(), torch.cat(pool.rows("v", lens)))


# ---------------------------------------------------------------------------- together
class Layer:
    """A decoder layer's attention block: norm, QKV, append, attention, quantizer, output projection."""

    def __init__(self, device, hidden=512, heads=4, kv_heads=2, dim=128, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        from oracle import reference
        rows = (heads + 2 * kv_heads) * dim
        qkv, qkv_s = reference.quantize_weight_128x128(torch.randn(rows, hidden, generator=g) * hidden ** -0.5)
        o, o_s = reference.quantize_weight_128x128(torch.randn(hidden, heads * dim, generator=g) * (heads * dim) ** -0.5)
        self.w = [t.to(device) for t in (qkv, qkv_s, o, o_s)]
        self.norm = (1 + 0.1 * torch.randn(hidden, generator=g)).to(BF16).to(device)

    def __call__(self, x, residual, cache, table, lens, indptr, rope):
        from tilegym_amd.suites.unsloth.ops import act_quant, w8a8_block_fp8_matmul
        q8, s8, residual = ops.rms_norm_quant(x, self.norm, 1e-5, residual=residual)
        qkv = w8a8_block_fp8_matmul(q8, self.w[0], s8, self.w[1], [128, 128], BF16).view(-1, self.heads + 2 * self.kv_heads, self.dim)
        q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], 1)
        q = ops.kv_cache_append(cache, k, v, table, lens, indptr, q=q, rope=rope)
        y = ops.kv_cache_attention(q, cache, table, lens, indptr)
        a8, a8_s = act_quant(y.view(y.shape[0], -1), 128)
        return w8a8_block_fp8_matmul(a8, self.w[2], a8_s, self.w[3], [128, 128], BF16), residual


def _whole(layer, x, residual, rope):
    """The layer over whole sequences in float64, nothing rounded but the weights, no cache."""
    qkv, qkv_s, o, o_s = (t.cpu().double() for t in layer.w)
    wide = lambda s, w: s.repeat_interleave(128, 0)[: w.shape[0]].repeat_interleave(128, 1)[:, : w.shape[1]]  # noqa: E731
    outs = []
    for xx, rr in zip(x, residual):
        _, y = R.ref_rms_norm(xx.cpu(), layer.norm.cpu(), 1e-5, rr.cpu())
        z = (y @ (qkv * wide(qkv_s, qkv)).t()).view(-1, layer.heads + 2 * layer.kv_heads, layer.dim)
        n = z.shape[0]
        z[:, : layer.heads + layer.kv_heads] = R.ref_rope(z[:, : layer.heads + layer.kv_heads], list(range(n)), rope, False)
        q, k, v = z.split([layer.heads, layer.kv_heads, layer.kv_heads], 1)
        out, _ = R.ref_attention(q, [k], [v], [n], [0, n], layer.dim ** -0.5)
        outs.append(out.reshape(n, -1) @ (o * wide(o_s, o)).t())
    return outs


@pytest.mark.gpu
def test_layer_in_chunks_and_in_a_graph(device):
    """Prompt, chunk, then single tokens replayed from a graph: near the layer in float64 over the whole sequences, and the
    replays the bits of the eager calls."""
    layer = Layer(device)
    total, chunks = [50, 37], [[30, 20], [13, 10], [1, 1], [1, 1], [1, 1], [1, 1], [1, 1], [1, 1], [1, 1]]
    g = torch.Generator().manual_seed(7)
    x = [torch.randn(n, 512, generator=g).to(BF16).to(device) for n in total]
    residual = [torch.randn(n, 512, generator=g).to(BF16).to(device) for n in total]
    rope = ops.rope_table(128, 128, device="cpu")
    want = _whole(layer, x, residual, rope)
    rope = rope.to(device)
    table = torch.tensor([[3, 0], [5, 1]], dtype=torch.int32, device=device)

    def run(graphs):
        cache, done, outs = ops.alloc_kv_cache(6, 2, 128, 64, device=device), [0, 0], [[], []]
        static = None
        for step, news in enumerate(chunks):
            xs = torch.cat([t[d:d + n] for t, d, n in zip(x, done, news)])
            rs = torch.cat([t[d:d + n] for t, d, n in zip(residual, done, news)])
            done = [d + n for d, n in zip(done, news)]
            lens = torch.tensor(done, dtype=torch.int32, device=device)
            indptr = torch.tensor([0] + list(itertools.accumulate(news)), dtype=torch.int32, device=device)
            if not graphs or step < 2:
                y, _ = layer(xs, rs, cache, table, lens, indptr, rope)
            else:
                if static is None:
                    static = {"x": xs.clone(), "r": rs.clone(), "lens": lens.clone(), "indptr": indptr.clone()}
                    side = torch.cuda.Stream()
                    side.wait_stream(torch.cuda.current_stream())
                    spare = ops.alloc_kv_cache(6, 2, 128, 64, device=device)
                    with torch.cuda.stream(side):
                        layer(static["x"], static["r"], spare, table, static["lens"], static["indptr"], rope)
                    torch.cuda.current_stream().wait_stream(side)
                    static["graph"] = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(static["graph"]):
                        static["y"], _ = layer(static["x"], static["r"], cache, table, static["lens"], static["indptr"], rope)
                static["x"].copy_(xs), static["r"].copy_(rs), static["lens"].copy_(lens)
                static["graph"].replay()
                torch.cuda.synchronize()
                y = static["y"].clone()
                torch.randn(1000, device=device).sum().item()  # the program's own work between replays
            at = 0
            for b, n in enumerate(news):
                outs[b].append(y[at:at + n])
                at += n
        return [torch.cat(o) for o in outs]

    eager, replayed = run(False), run(True)
    for b, n in enumerate(total):
        m = sum(c[b] for c in chunks)
        assert torch.equal(eager[b], replayed[b])
        got, ref = eager[b].cpu().double(), want[b][:m]
        # five roundings to e4m3 in a chain (activations, k, v, activations; the weights' are in the reference), each of a relative 2^-5 at the
        # root of the mean square at most, uncorrelated over 512 terms and more: 2^-5 * sqrt(5) < 0.07 of the result's size
        assert float((got - ref).norm() / ref.norm()) < 0.07


@pytest.mark.gpu
def test_two_graphs_share_no_scratch_memory(device):
    """Two attention calls whose contexts are split, captured on one stream, replayed at the same time on two."""
    pool = Pool(device, 130, 1, 64, 128, 2, 64)
    pool.fill([4000, 3900], [4000, 3900])
    q = [torch.randn(2, 8, 128, generator=pool.g).to(BF16).to(device) for _ in range(2)]
    args = (pool.cache, pool.i32(pool.table), pool.i32([4000, 3900]), pool.i32([0, 1, 2]))
    want = [ops.kv_cache_attention(x, *args) for x in q]
    assert _lib.load().tg_fp8_kv_attention_workspace_bytes(2, 8, 2, 1, 128, 64, 64, 0, 0) > 0
    graphs, outs = [], []
    for x in q:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.kv_cache_attention(x, *args))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in q]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


# ---------------------------------------------------------------------------- the forms that a call's sizes choose between
def test_table_beyond_the_positions_is_refused_without_a_device():
    a = {**_cache_args(page=128, batch=1), "table": torch.zeros(1, (1 << 23) + 1, dtype=torch.int32)}
    assert _attention_rc(a) == -6 and _read_rc(a) == -6 and _append_rc({**a, "rope": None, "q": None, "out": None}) == -6


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [33, 64, 70])
@pytest.mark.parametrize("dim,heads", [(128, 8), (64, 9), (256, 10)])
def test_attention_more_sequences_than_compute_units(device, batch, dim, heads):
    """Whole sequences of very different lengths, some of them equal, empty or without new tokens; then one with many more rows than a tile."""
    g = torch.Generator().manual_seed(batch)
    lens = torch.randint(0, 150, (batch,), generator=g).tolist()
    lens[3] = lens[4] = lens[-1] = 77
    lens[5] = 0
    news = [0 if n == 0 or b % 9 == 8 else 1 for b, n in enumerate(lens)]
    pool = Pool(device, batch * 3, heads, 64, dim, batch, 3)
    pool.fill(lens, lens)
    _attend(pool, lens, news, 2, BF16)
    lens[7], news[7] = 90, 21
    pool.fill([90 if b == 7 else 0 for b in range(batch)], [90 if b == 7 else 0 for b in range(batch)])
    _attend(pool, lens, news, 2, BF16)
    _attend(pool, lens, news, 2, BF16, window=30, sinks=2)


@pytest.mark.gpu
@pytest.mark.parametrize("page,dim", [(16, 64), (32, 128), (64, 128), (128, 64), (64, 256), (128, 256), (16, 256)])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("group,news", [(1, [1, 1]), (4, [4, 4]), (5, [5, 4]), (2, [70, 0]), (3, [150, 100])])
def test_attention_split_contexts(device, page, dim, dtype, group, news):
    """Every form of tile with its keys split over workgroups and joined."""
    lens = [1700, 1100]
    width = -(-2048 // page)
    pool = Pool(device, 2 * width, 1, page, dim, 2, width)
    pool.fill(lens, lens, dtype)
    assert _lib.load().tg_fp8_kv_attention_workspace_bytes(sum(news), group, 2, 1, dim, page, width, 0, 0) > 0
    _attend(pool, lens, news, group, dtype)
    _attend(pool, lens, news, group, dtype, window=1100, sinks=130)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 64])
def test_attention_many_sequences_of_many_rows(device, page):
    """More sequences than one prefix sum covers, each with more rows than a tile, a few with none."""
    batch = 140
    lens = [(7 * b) % 61 for b in range(batch)]
    news = [max(0, n - 5) for n in lens]
    width = -(-61 // page)
    pool = Pool(device, batch * width, 1, page, 64, batch, width)
    pool.fill(lens, lens)
    _attend(pool, lens, news, 6, BF16)


@pytest.mark.gpu
@pytest.mark.parametrize("page,dim,heads", CACHES)
def test_append_single_tokens_beside_a_chunk(device, page, dim, heads):
    """Mostly one token a sequence, and one sequence with a chunk over a page's border: a wave writes each page."""
    batch, chunk = 24, page + 19
    pool = Pool(device, batch * 3, heads, page, dim, batch, 3)
    rope = ops.rope_table(3 * page, dim, device="cpu")
    lens = [(5 * b) % page for b in range(batch)]
    pool.fill(lens, lens)
    news = [1] * batch
    news[2], news[11] = min(chunk, 4 * batch - 2 * batch), 0
    lens = [a + b for a, b in zip(lens, news)]
    assert sum(news) <= 4 * batch
    pool.fill(lens, news, BF16, rope)
    pool.check(True)


@pytest.mark.gpu
def test_call_paths_agree_and_refuse_alike(device, monkeypatch):
    """The native and the ctypes path: the same bits, the same refusals of tensors elsewhere and of values out of range."""
    lens, news = [100, 40], [3, 2]
    pool = Pool(device, 8, 2, 64, 128, 2, 2)
    pool.fill(lens, lens)
    qkv = torch.randn(5, 8, 128, generator=pool.g).to(BF16).to(device)
    q, k, v = qkv.split([4, 2, 2], 1)
    rope = ops.rope_table(128, 64, device=device)
    table, lens, indptr = pool.i32(pool.table), pool.i32(lens), pool.i32([0, 3, 5])
    x, w = torch.randn(5, 256, generator=pool.g).to(BF16).to(device), torch.ones(256, dtype=BF16, device=device)

    def run():
        cache = ops.KVCache(*(t.clone() for t in pool.cache))
        out = [ops.kv_cache_append(cache, k, v, table, lens, indptr, q=q, rope=rope), *cache]
        out += [ops.kv_cache_attention(q, cache, table, lens, indptr), *ops.kv_cache_read(cache, table, indptr, 5), *ops.rms_norm_quant(x, w)]
        errors = []
        for call in (lambda: ops.kv_cache_append(cache, k, v.cpu(), table, lens, indptr), lambda: ops.kv_cache_append(cache, k, v, table, lens, indptr.cpu()),
                     lambda: ops.kv_cache_append(cache, k, v, table, lens, indptr, q=q), lambda: ops.kv_cache_attention(q, cache, table.cpu(), lens, indptr),
                     lambda: ops.kv_cache_attention(q, cache, table, lens, indptr, window=2 ** 31),
                     lambda: ops.kv_cache_attention(q, cache, table, lens, indptr, window=4, sink_tokens=2 ** 31),
                     lambda: ops.kv_cache_attention(q, cache, table, lens, indptr, sink_tokens=-1),
                     lambda: ops.kv_cache_attention(q, cache, table, lens, indptr, out=torch.empty(5, 4, 128, dtype=BF16)),
                     lambda: ops.kv_cache_read(cache, table.cpu(), indptr, 5), lambda: ops.rms_norm_quant(x, w.cpu())):
            with pytest.raises(ValueError) as info:
                call()
            errors.append(str(info.value))
        for call in (lambda: ops.kv_cache_attention(q[:, :3], cache, table, lens, indptr), lambda: ops.kv_cache_attention(q, cache, table.long(), lens, indptr),
                     lambda: ops.kv_cache_append(cache, k[..., ::2], v, table, lens, indptr), lambda: ops.kv_cache_attention(q, cache, table, lens, indptr, sink_tokens=3),
                     lambda: ops.kv_cache_append(cache, k, v, table, lens, indptr, rope=rope[:127])):
            with pytest.raises(_lib.TileGymHipError) as info:
                call()
            errors.append(str(info.value))
        return out, errors

    native, said = run()
    monkeypatch.setattr(_lib, "native_path", lambda: False)
    plain, said_too = run()
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(native, plain))
    assert said == said_too


@pytest.mark.gpu
def test_calls_at_once_on_two_streams(device):
    """Split contexts, appends to caches of their own and norms on two streams, each twenty times over: the bits of the calls one by one."""
    pool = Pool(device, 130, 2, 64, 128, 2, 64)
    pool.fill([4000, 3900], [4000, 3900])
    table, lens, indptr = pool.i32(pool.table), pool.i32([4000, 3900]), pool.i32([0, 1, 2])
    qkv = [torch.randn(2, 12, 128, generator=pool.g).to(BF16).to(device) for _ in range(2)]
    x = [torch.randn(600, 1040, generator=pool.g).to(BF16).to(device) for _ in range(2)]
    w = torch.ones(1040, dtype=BF16, device=device)
    caches = [ops.KVCache(*(t.clone() for t in pool.cache)) for _ in range(2)]

    def step(i):
        q, k, v = qkv[i].split([8, 2, 2], 1)
        ops.kv_cache_append(caches[i], k, v, table, lens, indptr)
        return (ops.kv_cache_attention(q, caches[i], table, lens, indptr), *ops.rms_norm_quant(x[i], w, group_size=16))

    want = [step(i) for i in range(2)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(i))
    torch.cuda.synchronize()
    for i in range(2):
        for outs in got[i]:
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(outs, want[i]))


@pytest.mark.gpu
@pytest.mark.parametrize("page,dim", [(64, 128), (128, 64), (32, 256), (128, 256)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_append_long_runs_into_few_pages(device, page, dim, dtype):
    """Few pages and many new tokens of each: from a page's beginning, then from the middle of one."""
    pool = Pool(device, 12, 2, page, dim, 2, 5)
    rope = ops.rope_table(5 * page, dim, device="cpu")
    lens = [2 * page + 5, page - 3]
    pool.fill(lens, lens, dtype, rope, True)
    pool.check(True)
    news = [2 * page + 1, 3 * page + 3]
    q, out, want, _ = pool.fill([a + b for a, b in zip(lens, news)], news, dtype, rope, True, q_heads=3)
    pool.check(True)
    slack = 2.0 ** -22 * 2 * want.abs().amax()  # two products and a difference in fp32
    assert bool(((out.cpu().double() - want).abs() <= HALF[dtype] * want.abs() * (1 + 2.0 ** -10) + slack + 2.0 ** -26).all())


# ---------------------------------------------------------------------------- values and arguments at the edges
@pytest.mark.gpu
@pytest.mark.parametrize("given", [False, True])
def test_norm_of_rows_next_to_nothing(device, given):
    """Scales below the smallest normal number: zeros stay zeros, the others are rounded as ever."""
    g = torch.Generator().manual_seed(5)
    x = torch.randn(6, 512, generator=g) * 1e-36
    x[:, ::3] = 0
    w = torch.full((512,), 1e-4)
    scale = torch.tensor([3e-40], device=device) if given else None
    q, s = ops.rms_norm_quant(x.to(device), w.to(device), 1e-6, group_size=128, scale=scale)
    y = x.double() * 1e3 * 1e-4  # (the mean square is nothing beside eps)
    step = (s.cpu().double() if not given else torch.full((6, 4), float(scale))).repeat_interleave(128, 1)
    got = q.cpu().float().double() * step
    assert bool((step < 2.0 ** -126).all()) and bool((got[:, ::3] == 0).all())
    # half an e4m3 step, and the fp32 steps below 2^-126: 2^-150 off for y, and as much relative to a scale of 2^-150 / scale
    y = torch.minimum(torch.maximum(y, -448 * step), 448 * step)
    assert bool(((got - y).abs() <= 2.0 ** -4 * y.abs() * (1 + 2.0 ** -10) + 2 * step * 2.0 ** -10 + 2.0 ** -149 + y.abs() * 2.0 ** -149 / step).all())


@pytest.mark.gpu
def test_norm_flags_that_are_not_bools(device):
    x, w = torch.randn(3, 128, device=device).to(BF16), torch.ones(128, dtype=BF16, device=device)
    want = ops.rms_norm_quant(x, w, return_norm=True)
    got = ops.rms_norm_quant(x, w, return_norm=1)
    assert len(got) == 3 and torch.equal(got[2], want[2]) and len(ops.rms_norm_quant(x, w, return_norm=0)) == 2


@pytest.mark.gpu
@pytest.mark.parametrize("news", [1, 24])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attention_many_faint_keys(device, dtype, news):
    """One strong key with value zero beside twenty thousand faint ones with value one, each 2^-25.2 of it."""
    n, dim, strong = 20000, 64, 20.0
    cache = ops.alloc_kv_cache(-(-n // 64), 1, dim, 64, device=device)
    k, v = torch.zeros(n, 1, dim), torch.ones(n, 1, dim)
    k[:, 0, 0] = 2.5
    k[0, 0, 0], v[0] = strong, 0
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    table = torch.arange(-(-n // 64), dtype=torch.int32, device=device)[None]
    ops.kv_cache_append(cache, k.to(dtype).to(device), v.to(dtype).to(device), table, i32(n), i32(0, n))
    q = torch.zeros(news, 4, dim)
    q[..., 0] = 1
    out = ops.kv_cache_attention(q.to(dtype).to(device), cache, table, i32(n), i32(0, news), sm_scale=1.0).cpu().double()
    weight = math.exp(2.5 - strong)
    for t in range(news):
        faint = n - news + t
        want = faint * weight / (1 + faint * weight)
        # a weight is rounded to 16 bits, or by half of f16's smallest step, a 128th of 2^-25 against the maximum; the scores' 20 are 2^-23 off, the
        # exponentials and the sum of 20000 fp32 terms a few units of 2^-24 each
        tol = want * (2 * HALF[dtype] + 20 * 2.0 ** -22 + 20000 / 16 * 2.0 ** -24) + (faint * 2.0 ** -32 if dtype == F16 else 0)
        assert bool(((out[t] - want).abs() <= tol).all()), (float(out[t, 0, 0]), want)


@pytest.mark.gpu
@pytest.mark.parametrize("news", [6, 40])
def test_attention_of_more_new_tokens_than_there_are_in_the_widest_window(device, news):
    """Positions below zero see nothing, whatever the window; those from zero on see all before them."""
    pool = Pool(device, 2, 1, 64, 64, 1, 1)
    pool.fill([3], [3])
    q = torch.randn(news, 4, 64, generator=pool.g).to(BF16).to(device)
    args = (q, pool.cache, pool.i32(pool.table), pool.i32([3]), pool.i32([0, news]))
    want = ops.kv_cache_attention(*args)
    assert bool((want[:news - 3] == 0).all()) and bool((want[news - 3:] != 0).any(-1).all())
    for window in (2 ** 31 - 1, 2 ** 31 - 3, 2 ** 30, 3):
        assert torch.equal(ops.kv_cache_attention(*args, window=window, sink_tokens=0), want)


@pytest.mark.gpu
def test_launches_too_large_for_the_device_are_refused(device):
    """Small tensors whose sequences and heads would make more work items than a launch can have."""
    heads = 65536
    cache = ops.alloc_kv_cache(1, heads, 64, 16, device=device)
    table, lens = torch.full((256, 1), -1, dtype=torch.int32, device=device), torch.zeros(256, dtype=torch.int32, device=device)
    indptr = torch.zeros(257, dtype=torch.int32, device=device)
    x = torch.zeros(1, heads, 64, dtype=BF16, device=device)
    for call in (lambda: ops.kv_cache_read(cache, table, indptr, 1), lambda: ops.kv_cache_append(cache, x, x, table, lens, indptr),
                 lambda: ops.kv_cache_attention(x, cache, table, lens, indptr)):
        with pytest.raises(_lib.TileGymHipError):
            call()
    # nothing is left behind: a smaller call of the same kind runs
    out = ops.kv_cache_attention(x, cache, table[:1], lens[:1], indptr[:2], out=torch.full_like(x, 3.0))
    assert bool((out == 3).all())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,hidden", [(600, 4112), (513, 5120), (777, 8192)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_norm_of_many_rows_of_two_vectors_a_lane(device, rows, hidden, dtype):
    """512 rows and more of 4097 to 8192 elements have a form of their own."""
    x, r, w = _norm_case(rows, hidden, dtype, device)
    *out, norm = ops.rms_norm_quant(x, w, 1e-5, residual=r, group_size=16, return_norm=True)
    _check_norm(out, x, w, 1e-5, r, 16, None, dtype)
    _, y = R.ref_rms_norm(x.cpu(), w.cpu(), 1e-5, r.cpu())
    # f16's numbers below 2^-14 are 2^-24 apart, so a rounding there is off by up to 2^-25, more than 2^-11 of the value; some of these 2.5 to 6
    # million elements are that small.  (bf16 and fp32 have nothing as coarse near zero.)
    smallest = 2.0 ** -25 if dtype == F16 else 0.0
    assert bool(((norm.cpu().double() - y).abs() <= (HALF[dtype] + 2.0 ** -18) * y.abs() + smallest + 2.0 ** -126).all())
    scale = torch.tensor([0.02], device=device)
    _check_norm(ops.rms_norm_quant(x, w, 1e-5, group_size=None, scale=scale), x, w, 1e-5, None, None, scale, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("page,dim,heads", CACHES)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_append_a_wave_per_page_over_a_border(device, page, dim, heads, dtype):
    """Mostly one token a sequence, and one sequence with a chunk that ends in a later page than it begins in; a wave writes each page."""
    batch, chunk = 24, 48
    pool = Pool(device, batch * 5, heads, page, dim, batch, 5)
    rope = ops.rope_table(5 * page, dim, device="cpu")
    lens = [(5 * b) % page for b in range(batch)]
    lens[2] = page - 5
    pool.fill(lens, lens, dtype)
    news = [1] * batch
    news[2], news[11] = chunk, 0
    assert sum(news) <= 4 * batch and (lens[2] + chunk - 1) // page > lens[2] // page
    pool.fill([a + b for a, b in zip(lens, news)], news, dtype, rope)
    pool.check(True)


# ---------------------------------------------------------------------------- torch's dispatcher
def test_operators_infer_shapes_through_torchs_dispatcher():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from tilegym_amd import torch_ops
    names = ("fp8_rms_norm_quant", "fp8_kv_append", "fp8_kv_append_turn", "fp8_kv_read", "fp8_kv_attention")
    assert {f"tilegym_hip::{n}" for n in names} <= set(torch_ops.registered_ops())
    t = torch.ops.tilegym_hip
    for op in (t.fp8_kv_append, t.fp8_kv_append_turn):  # the cache's four tensors are written, nothing else is
        assert [a.name for a in op.default._schema.arguments if a.alias_info is not None and a.alias_info.is_write] == ["k_cache", "v_cache", "k_scale", "v_scale"]
    with FakeTensorMode(allow_non_fake_inputs=True):
        e = lambda *s, dtype=BF16: torch.empty(*s, dtype=dtype, device="cuda")  # noqa: E731
        got = t.fp8_rms_norm_quant(e(4, 3, 256), e(256), 1e-6, e(4, 3, 256), 64, None, True)
        assert [(tuple(x.shape), x.dtype) for x in got] == [((4, 3, 256), FP8), ((4, 3, 4), F32), ((4, 3, 256), BF16), ((4, 3, 256), BF16)]
        assert len(t.fp8_rms_norm_quant(e(4, 256), e(256), 1e-6, None, 0, e(1, dtype=F32), False)) == 1
        with pytest.raises(ValueError):
            t.fp8_rms_norm_quant(e(4, 240), e(240), 1e-6, None, 128, None, False)
        i32 = lambda *s: e(*s, dtype=torch.int32)  # noqa: E731
        cache = (e(9, 2, 64, 128, dtype=FP8), e(9, 2, 128, 64, dtype=FP8), e(9, 2, dtype=F32), e(9, 2, dtype=F32))
        batch, rope = (i32(3, 4), i32(3), i32(4)), e(256, 64, dtype=F32)
        assert t.fp8_kv_append(*cache, e(5, 2, 128), e(5, 2, 128), *batch, rope, False) is None
        q = t.fp8_kv_append_turn(*cache, e(5, 2, 128), e(5, 2, 128), *batch, e(5, 12, 128)[:, :8], rope, True)
        assert q.shape == (5, 8, 128) and q.is_contiguous()
        k, v = t.fp8_kv_read(*cache, batch[0], batch[2], 77, F32)
        assert k.shape == v.shape == (77, 2, 128) and k.dtype == F32
        out = t.fp8_kv_attention(e(5, 12, 128)[:, :8], *cache, *batch, None, 0, 0)
        assert out.shape == (5, 8, 128) and out.is_contiguous() and out.dtype == BF16
        with pytest.raises(ValueError):
            t.fp8_kv_attention(e(5, 8, 64), *cache, *batch, None, 0, 0)
    x = torch.zeros(2, 128)
    with pytest.raises(NotImplementedError):
        t.fp8_rms_norm_quant(x, x[0], 1e-6, None, 128, None, False)


@pytest.mark.gpu
def test_operators_through_torchs_dispatcher(device):
    """The bits of the direct calls, one by one and in a graph traced whole, caches written in place."""
    lens, news = [100, 40], [3, 2]
    pool = Pool(device, 8, 2, 64, 128, 2, 2)
    pool.fill(lens, lens)
    x, r = (torch.randn(5, 1024, generator=pool.g).to(BF16).to(device) for _ in range(2))
    w, rope, scale = torch.ones(1024, dtype=BF16, device=device), ops.rope_table(128, 64, device=device), torch.tensor([0.02], device=device)
    batch = (pool.i32(pool.table), pool.i32(lens), pool.i32([0, 3, 5]))
    bits = lambda ts: [t.view(torch.uint8).clone() for t in ts]  # noqa: E731

    def direct(cache):
        norm = ops.rms_norm_quant(x, w, 1e-5, residual=r, return_norm=True)
        q, k, v = norm[3].view(5, 8, 128).split([4, 2, 2], 1)
        turned = ops.kv_cache_append(cache, k, v, *batch, q=q, rope=rope)
        ops.kv_cache_append(cache, k, v, *batch)
        out = ops.kv_cache_attention(turned, cache, *batch, window=50, sink_tokens=2)
        return [*norm, *ops.rms_norm_quant(x, w, 1e-5, scale=scale)[:1], turned, out, *ops.kv_cache_read(cache, batch[0], batch[2], 5, F32)]

    def through(c0, c1, c2, c3, x, w, r, scale, table, lens, indptr, rope):
        t, c, b = torch.ops.tilegym_hip, (c0, c1, c2, c3), (table, lens, indptr)
        norm = t.fp8_rms_norm_quant(x, w, 1e-5, r, 128, None, True)
        q, k, v = norm[3].view(5, 8, 128).split([4, 2, 2], 1)
        turned = t.fp8_kv_append_turn(*c, k, v, *b, q, rope, False)
        t.fp8_kv_append(*c, k, v, *b, None, False)
        out = t.fp8_kv_attention(turned, *c, *b, None, 50, 2)
        return [*norm, *t.fp8_rms_norm_quant(x, w, 1e-5, None, 0, scale, False), turned, out, *t.fp8_kv_read(c[0], c[1], c[2], c[3], b[0], b[2], 5, F32)]

    cache = ops.KVCache(*(t.clone() for t in pool.cache))
    want = bits(direct(cache)) + bits(cache)
    for call in (through, torch.compile(through, backend="aot_eager", fullgraph=True)):
        cache = ops.KVCache(*(t.clone() for t in pool.cache))
        got = bits(call(*cache, x, w, r, scale, *batch, rope)) + bits(cache)
        assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("hidden", [512, 4096, 8192, 16384])
def test_norm_codes_are_those_of_the_quantizer(device, hidden):
    """With fp32 rows, which come out unrounded: scales and codes are the bits of act_quant on them, every division included."""
    from tilegym_amd.suites.unsloth.ops import act_quant
    g = torch.Generator(device=device).manual_seed(hidden)
    x = torch.randn((1 << 25) // hidden, hidden, generator=g, device=device)
    w = 1 + 0.2 * torch.randn(hidden, generator=g, device=device)
    for group in (16, 128):
        q, scales, norm = ops.rms_norm_quant(x, w, 1e-5, group_size=group, return_norm=True)
        want, want_scales = act_quant(norm, group)
        assert torch.equal(scales, want_scales) and torch.equal(q.view(torch.uint8), want.view(torch.uint8))
    # a given scale: the IEEE quotient, cut and rounded
    for s in (0.03, 0.0123):
        scale = torch.tensor([s], device=device)
        q, _, norm = ops.rms_norm_quant(x, w, 1e-5, scale=scale, return_norm=True)
        assert torch.equal(q.view(torch.uint8), (norm / scale).clamp(-448, 448).to(FP8).view(torch.uint8))


@pytest.mark.gpu
@pytest.mark.parametrize("given", [1e-30, 1e-17, 0.02, 3e18, 1e30])
def test_norm_with_a_given_scale_saturates(device, given):
    """Infinite and very large elements against small, ordinary and large scales: +-448 by their sign, NaN -448, zeros zero."""
    x = torch.tensor([1.0, -1.0, 0.0, -0.0] * 128).repeat(4, 1)
    w = torch.tensor([math.inf, 3e38, 1e30, 1.0, 1e-30, 0.0, math.nan, -math.inf]).repeat_interleave(64)
    scale = torch.tensor([given], device=device)
    q, _, norm = ops.rms_norm_quant(x.to(device), w.to(device), 0.0, scale=scale, return_norm=True)
    y = norm.cpu()
    want = (y / given).clamp(-448, 448)
    want = torch.where(torch.isnan(want), torch.full_like(want, -448.0), want).to(FP8)
    assert torch.equal(q.cpu().float(), want.float())


@pytest.mark.gpu
def test_append_turns_q_of_positions_outside_the_table_by_its_ends(device):
    """More new tokens than the sequence has, and a length beyond the table: finite rows, by the first and the last angles."""
    pool = Pool(device, 4, 1, 16, 64, 2, 2)
    rope = ops.rope_table(32, 64, base=50.0, device="cpu")
    k = torch.randn(9, 1, 64, generator=pool.g).to(BF16).to(device)
    q = torch.randn(9, 3, 64, generator=pool.g).to(BF16)
    out = ops.kv_cache_append(pool.cache, k, k, pool.i32(pool.table), pool.i32([2, 34]), pool.i32([0, 5, 9]), q=q.to(device), rope=rope.to(device))
    want = R.ref_rope(q, [0, 0, 0, 0, 1, 30, 31, 31, 31], rope, False)
    # one rounding to bf16, and two products and a difference in fp32
    assert bool(((out.cpu().double() - want).abs() <= 2.0 ** -8 * (1 + 2.0 ** -10) * want.abs() + 2.0 ** -21 * want.abs().amax()).all())
