"""Tokens carried by ``moe_sort`` and ``moe_permute`` to the segments of ``ragged_block_scaled_bmm`` and back: a layer's FP8 projection over experts, as a program puts it together."""

import pytest
import torch

from tilegym_amd import ops
from tilegym_amd.quant import act_quant
from tilegym_amd.suites.flashinfer.ops import ragged_block_scaled_bmm

from .test_int8_ops import BF16, F16, HALF, TINY, gen, routing


def _weights(experts, n, k, seed):
    b = (0.5 * torch.randn(experts, n, k, generator=gen(seed))).clamp(-448, 448).to(torch.float8_e4m3fn)
    return b, 0.01 * torch.exp(torch.randn(experts, (n + 127) // 128, k // 128, generator=gen(seed + 1)))


def _unscaled(q, s):
    return q.double() * s.double().repeat_interleave(128, -1)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,experts,k,h,n,absent,dtype", [(1, 4, 2, 128, 256, False, BF16), (37, 8, 3, 256, 384, True, BF16), (300, 16, 4, 512, 256, True, F16),
                                                              (1500, 64, 6, 256, 640, False, BF16)])
def test_projection_over_experts(device, tokens, experts, k, h, n, absent, dtype):
    ids, x = routing(tokens, experts, k, 1, absent=absent), torch.randn(tokens, h, generator=gen(2)).to(dtype)
    b, b_s = _weights(experts, n, h, 3)
    w = torch.rand(tokens, k, generator=gen(5))
    order = ops.moe_sort(ids.to(device), experts)
    # quantized in the experts' order; the reference quantizes the tokens: a row's codes are its own
    rows = ops.moe_permute(x.to(device), order)
    a, a_s = act_quant(rows)
    y = torch.zeros(tokens * k, n, dtype=dtype, device=device)
    made = ragged_block_scaled_bmm(a, b.to(device), a_s, b_s.to(device), order.indptr, tokens, out_dtype=dtype)
    live = int(order.indptr[-1])
    assert made.shape == y.shape
    y[:live] = made[:live]
    out = ops.moe_unpermute(y, order, w.to(device)).cpu().double()

    q, s = act_quant(x.to(device))
    x64, slots = _unscaled(q.cpu(), s.cpu()), order.slots.cpu().long()
    exact, size = torch.zeros(tokens, n, dtype=torch.float64), torch.zeros(tokens, n, dtype=torch.float64)
    off = torch.zeros(tokens, n, dtype=torch.float64)
    for e in range(experts):
        token, slot = torch.nonzero(ids.long() == e, as_tuple=True)
        if not token.numel():
            continue
        b64 = (b[e].double() * b_s[e].double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1))
        made64, made_size, weight = x64[token] @ b64.t(), x64[token].abs() @ b64.abs().t(), w[token, slot].double()[:, None]
        # a row: its products (exact) summed in fp32 with a block's two scales, at most two roundings each, and rounded to the type
        row_off = (2 * h + 8) * 2.0 ** -24 * made_size + HALF[dtype] * made64.abs() + TINY[dtype]
        exact.index_add_(0, token, weight * made64)
        size.index_add_(0, token, weight * made64.abs())
        off.index_add_(0, token, weight * 1.01 * row_off)
        first = int(order.indptr[e])
        assert torch.equal(slots[first:first + token.numel()], (token * k + slot))
    # the weighted sum: a product and an addition a slot, and the store's
    tol = off + (2 * k * 2.0 ** -24 + HALF[dtype]) * 1.01 * (size + off) + TINY[dtype]
    assert bool(((out - exact).abs() <= tol).all()), float(((out - exact).abs() / tol).max())
    assert not bool(out[(order.rows.cpu() < 0).all(1)].any())
