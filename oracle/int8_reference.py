"""Oracle of the products in 8-bit integers and of the ways to the experts and back: float64 on the CPU, loops where they are plainest.  Test
infrastructure."""

from __future__ import annotations

import torch


def ref_int8_matmul(a, b, scale_a, scale_b, bias=None):
    """(the result, |scales * sum|) in float64; the sum itself is exact in int64."""
    total = (a.cpu().long() @ b.cpu().long().t()).double()
    part = total * scale_a.cpu().double().reshape(-1, 1) * scale_b.cpu().double().reshape(1, -1)
    return (part if bias is None else part + bias.cpu().double()), part.abs()


def ref_int8_matmul_f32(a, b, scale_a, scale_b):
    """Without a bias, in the kernels' fp32 steps: float(sum), times the token's scale, times the channel's."""
    total = a.cpu().long() @ b.cpu().long().t()
    return total.float() * scale_a.cpu().reshape(-1, 1) * scale_b.cpu().reshape(1, -1)


def ref_ragged(a, b, scale_a, scale_b, indptr, fn):
    """fn of each expert's rows, one after the other; rows of no expert are NaN."""
    out = torch.full((a.shape[0], b.shape[1]), float("nan"), dtype=torch.float64)
    ends = indptr.tolist()
    for e, (lo, hi) in enumerate(zip(ends, ends[1:])):
        if hi > lo:
            got = fn(a[lo:hi], b[e], scale_a.reshape(-1)[lo:hi] if scale_a.numel() > 1 else scale_a, scale_b[e] if scale_b.numel() > 1 else scale_b)
            out[lo:hi] = (got[0] if isinstance(got, tuple) else got).double()
    return out


def ref_quant(x):
    """The fp32 steps of quant_int8 (the CPU's products, division and rounding)."""
    x = x.cpu().float()
    amax = x.abs().amax(-1) if x.shape[-1] else x.new_zeros(x.shape[:-1])
    scale = amax * torch.tensor(1 / 127, dtype=torch.float32)
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    bad = ~torch.isfinite(x).all(-1)
    q = (x / scale[..., None]).round().clamp(-127, 127)
    q = torch.where(bad[..., None], torch.zeros_like(q), q)
    return q.to(torch.int8), torch.where(bad, torch.full_like(scale, float("nan")), scale)


def ref_sort(ids, experts):
    """(indptr, rows, slots) as lists, by buckets."""
    flat = ids.flatten().tolist()
    buckets = [[] for _ in range(experts + 1)]
    for slot, e in enumerate(flat):
        buckets[e if 0 <= e < experts else experts].append(slot)
    slots, indptr = [], []
    for bucket in buckets:
        indptr.append(len(slots))
        slots += bucket
    rows = [0] * len(flat)
    for row, slot in enumerate(slots):
        rows[slot] = row if row < indptr[-1] else -1 - row
    return indptr, rows, slots


def ref_permute(x, rows):
    x, out = x.cpu().double(), torch.zeros(rows.numel(), x.shape[1], dtype=torch.float64)
    for t, places in enumerate(rows.tolist()):
        for r in places:
            if r >= 0:
                out[r] = x[t]
    return out


def ref_unpermute(x, rows, weights=None):
    """(the result, sum |weight * x|) in float64."""
    x = x.cpu().double()
    out, size = (torch.zeros(rows.shape[0], x.shape[1], dtype=torch.float64) for _ in range(2))
    for t, places in enumerate(rows.tolist()):
        for j, r in enumerate(places):
            if r >= 0:
                v = x[r] * (1.0 if weights is None else float(weights[t, j]))
                out[t] += v
                size[t] += v.abs()
    return out, size


def ref_unpermute_backward(grad, x, rows, weights):
    """(grad_x, grad_weights, sum |grad * x| of each weight's) in float64."""
    grad, x = grad.cpu().double(), x.cpu().double()
    gx, gw, size = torch.zeros_like(x), torch.zeros(rows.shape, dtype=torch.float64), torch.zeros(rows.shape, dtype=torch.float64)
    for t, places in enumerate(rows.tolist()):
        for j, r in enumerate(places):
            if r >= 0:
                gx[r] = float(weights[t, j]) * grad[t]
                gw[t, j] = (grad[t] * x[r]).sum()
                size[t, j] = (grad[t] * x[r]).abs().sum()
    return gx, gw, size
