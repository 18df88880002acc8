"""The operators around a decoder layer's FP8 projections in float64, written from their definitions -- TEST INFRASTRUCTURE ONLY.

Sequence by sequence, page by page, on the CPU.  Nothing of the product is imported here."""

from __future__ import annotations

import math
from typing import List, Optional, Sequence, Tuple

import torch

FP8 = torch.float8_e4m3fn
MAX = 448.0


def ref_rms_norm(x, weight, eps, residual=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(x + residual, its norm times weight)."""
    s = x.double() if residual is None else x.double() + residual.double()
    return s, s / torch.sqrt(s.pow(2).mean(-1, keepdim=True) + eps) * weight.double()


def ref_group_scales(y: torch.Tensor, group: int) -> torch.Tensor:
    s = y.reshape(*y.shape[:-1], -1, group).abs().amax(-1) / MAX
    return torch.where(s == 0, torch.ones_like(s), s)


def ref_rope(x: torch.Tensor, positions: Sequence[int], table: torch.Tensor, interleaved: bool) -> torch.Tensor:
    """x (tokens, heads, D) with its first table.shape[1] elements turned."""
    out, r = x.double().clone(), table.shape[1]
    for t, p in enumerate(positions):
        cos, sin = table[p, : r // 2].double(), table[p, r // 2:].double()
        for i in range(r // 2):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
            out[t, :, a] = x[t, :, a].double() * cos[i] - x[t, :, b].double() * sin[i]
            out[t, :, b] = x[t, :, a].double() * sin[i] + x[t, :, b].double() * cos[i]
    return out


def ref_page_scale(amax: float) -> float:
    """2^e with the smallest e in [-40, 40] for which amax <= 448 * 2^e."""
    e = -40
    while e < 40 and amax > MAX * 2.0 ** e:
        e += 1
    return 2.0 ** e


class RefCache:
    """What a paged cache should hold: each written slot's exact element, and each page's scale."""

    def __init__(self, pages: int, heads: int, page: int, dim: int):
        self.page, self.shape = page, (pages, heads, page, dim)
        self.value = {n: torch.full(self.shape, math.nan, dtype=torch.float64) for n in ("k", "v")}
        self.scale = {n: torch.ones(pages, heads, dtype=torch.float64) for n in ("k", "v")}

    def append(self, k, v, table, lens, indptr) -> None:
        """k, v: (tokens, heads, D) as they are to be written (turned already)."""
        for b, length in enumerate(lens):
            n = indptr[b + 1] - indptr[b]
            start = length - n
            first = max(start, 0)
            for begin in range(first // self.page * self.page, length, self.page):
                index = begin // self.page
                if index >= len(table[b]) or not 0 <= table[b][index] < self.shape[0]:
                    continue
                page, lo, hi = table[b][index], max(begin, first), min(begin + self.page, length)
                for name, x in (("k", k), ("v", v)):
                    new = x[indptr[b] + lo - start: indptr[b] + hi - start].double()
                    for h in range(self.shape[1]):
                        finite = new[:, h][~torch.isnan(new[:, h])]
                        s = ref_page_scale(float(finite.abs().max()) if finite.numel() else 0.0)
                        if lo > begin:
                            s = max(s, float(self.scale[name][page, h]))
                        self.scale[name][page, h] = s
                        self.value[name][page, h, lo - begin: hi - begin] = new[:, h]


def ref_attention(q, k: List[torch.Tensor], v: List[torch.Tensor], lens, indptr, scale: float, window: int = 0, sinks: int = 0,
                  half_step: float = 0.0, v_unit: float = 0.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(out, how far a kernel may be off) per element.  k[b], v[b]: (positions, heads, D) of sequence b; what no token sees may be anything.

    The bound: the weights are rounded once to 16 bits (half_step of each, so half_step * sum p |v|), a score is a sum of D products
    in fp32 (an error of at most D 2^-24 sum |q k| each way moves its weight by as much, and the sum of weights too), the exponential and
    the running rescales cost a few units of 2^-24 per step of keys; the result is rounded once (half_step * |out|).  In f16
    a weight under 2^-14 is off by up to 2^-25 whatever its size, times a value of up to 448 of the largest scale (v_unit)."""
    out = torch.zeros(q.shape, dtype=torch.float64)
    tol = torch.zeros(q.shape, dtype=torch.float64)
    group = q.shape[1] // (k[0].shape[1] if k else 1)
    for b, length in enumerate(lens):
        n = indptr[b + 1] - indptr[b]
        for t in range(n):
            p = length - n + t
            seen = [j for j in range(min(p + 1, k[b].shape[0])) if not window or p - j < window or j < sinks]
            if not seen:
                continue
            kk, vv = k[b][seen].double(), v[b][seen].double()
            for h in range(q.shape[1]):
                qq = q[indptr[b] + t, h].double()
                s = kk[:, h // group] @ qq * scale
                w = torch.softmax(s, 0)
                row = indptr[b] + t
                out[row, h] = w @ vv[:, h // group]
                size = w @ vv[:, h // group].abs()
                spread = float((kk[:, h // group].abs() @ qq.abs()).max()) * abs(scale)
                fp32 = 2 * (q.shape[2] + 8) * 2.0 ** -24 * spread + (8 + len(seen) / 16) * 2.0 ** -23
                tol[row, h] = (half_step + fp32) * size * 1.01 + half_step * out[row, h].abs()
                if half_step < 2.0 ** -9:
                    tol[row, h] += len(seen) * 2.0 ** -25 * 448 * v_unit
    return out, tol + 1e-30


def ref_attention_by_head(q, k: List[torch.Tensor], v: List[torch.Tensor], lens, indptr, scale: float, window: int = 0, sinks: int = 0,
                          half_step: float = 0.0, v_scale: Optional[List[torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """ref_attention with a head's rows of a sequence in one product, on the tensors' device; v_scale[b] (positions, heads): the scale that
    each value's code is multiplied by.

    Two terms of the bound are its own.  A weight times its value's scale is an exponential whose argument holds the scale's logarithm: off by
    2^-24 of that twice.  And in f16 a weight is off by up to half of the smallest step, 2^-25, where the row's largest product of weight and scale stands
    at 2^7 at least: 2^-32 of that product, times a code of up to 448, for each key; a result is off by 2^-25 below 2^-14."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    group, f16 = q.shape[1] // (k[0].shape[1] if k else 1), 0 < half_step < 2.0 ** -9
    for b, length in enumerate(lens):
        n = indptr[b + 1] - indptr[b]
        if n == 0 or k[b].shape[0] == 0:
            continue
        p = torch.arange(length - n, length, device=q.device)[:, None]
        j = torch.arange(k[b].shape[0], device=q.device)[None, :]
        seen = j <= p
        if window:
            seen = seen & ((p - j < window) | (j < sinks))
        some = seen.any(1, keepdim=True)
        count = seen.sum(1, keepdim=True).double()
        rows = slice(indptr[b], indptr[b] + n)
        for h in range(q.shape[1]):
            kk, vv, qq = k[b][:, h // group].double(), v[b][:, h // group].double(), q[rows, h].double()
            s = (qq @ kk.t()) * scale
            w = torch.where(some, torch.softmax(s.masked_fill(~seen & some, -math.inf), 1) * seen, torch.zeros_like(s))
            out[rows, h] = w @ vv
            spread = ((qq.abs() @ kk.abs().t()) * seen).amax(1, keepdim=True) * abs(scale)
            units = torch.ones(kk.shape[0], dtype=torch.float64, device=q.device) if v_scale is None else v_scale[b][:, h // group].double()
            binades = float(units.log2().abs().max())
            fp32 = 2 * (q.shape[2] + 8) * 2.0 ** -24 * spread + (8 + count / 16 + binades) * 2.0 ** -23
            tol[rows, h] = (half_step + fp32) * (w @ vv.abs()) * 1.01 + half_step * out[rows, h].abs()
            if f16:
                tol[rows, h] += count * 2.0 ** -32 * 448 * (w * units).amax(1, keepdim=True) + 2.0 ** -25
    return out, tol + 1e-30
