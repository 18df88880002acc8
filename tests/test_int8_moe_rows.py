"""The type that int8_moe holds its second product's rows in."""

import pytest
import torch

from oracle import int8_reference as R
from tilegym_amd import _lib, ops

from .test_int8_ops import BF16, F16, F32, HALF, TINY, bits, codes, gen, routing, scales


def test_other_types_are_refused():
    x, w = torch.zeros(2, 64, dtype=BF16), torch.zeros(1, 64, 64, dtype=torch.int8)
    one, ids = torch.ones(1), torch.zeros(2, 1, dtype=torch.int32)
    for t in (F16, torch.float64, torch.int8):
        with pytest.raises(ValueError, match="rows_dtype"):
            ops.int8_moe(x, w, w[:, :, :32].contiguous(), one, one, torch.ones(2, 1), ids, rows_dtype=t)
    for t in (None, BF16, F32):
        with pytest.raises(RuntimeError, match="HIP device"):
            ops.int8_moe(x, w, w[:, :, :32].contiguous(), one, one, torch.ones(2, 1), ids, rows_dtype=t)


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("tokens,experts,k,h,i,dtype", [(1, 4, 2, 64, 32, BF16), (9, 64, 6, 256, 100, F16), (33, 8, 2, 250, 64, BF16), (700, 16, 4, 512, 192, BF16), (0, 4, 2, 64, 32, BF16)])
def test_rows_in_float32(device, monkeypatch, native, tokens, experts, k, h, i, dtype):
    """Against the weighted sum of the same codes' products in 64 bits: one rounding to the type, and fp32's."""
    if not native:
        monkeypatch.setattr(_lib, "native_path", lambda: False)
    x = torch.randn(tokens, h, generator=gen(1)).to(dtype).to(device)
    w1, w2 = codes((experts, 2 * i, h), 2).to(device), codes((experts, h, i), 3).to(device)
    s1, s2 = scales((experts, 2 * i), 4).to(device) / 50, scales((experts, h), 5).to(device)
    ids, w = routing(tokens, experts, k, 6, absent=True).to(device), torch.rand(tokens, k, generator=gen(7)).to(device)
    got = ops.int8_moe(x, w1, w2, s1, s2, w, ids, rows_dtype=F32)
    assert got.shape == x.shape and got.dtype == dtype and not got.requires_grad
    assert torch.equal(bits(ops.int8_moe(x, w1, w2, s1, s2, w, ids, rows_dtype=dtype)), bits(ops.int8_moe(x, w1, w2, s1, s2, w, ids)))
    order = ops.moe_sort(ids, experts)
    q, s = ops.moe_permute_quant_int8(x, order)
    q, s = ops.silu_mul_quant_int8(ops.ragged_int8_matmul(q, w1, s, s1, order.indptr, out_dtype=dtype))
    ptr, rows, y = order.indptr.tolist(), order.rows.cpu(), torch.zeros(tokens * k, h, dtype=torch.float64)
    for e in range(experts):
        part = slice(ptr[e], ptr[e + 1])
        y[part] = R.ref_int8_matmul(q[part], w2[e], s[part], s2[e])[0]
    exact, size = R.ref_unpermute(y, rows, w)
    # a row: the sum's conversion and two products; a slot: a product and an addition; the rounding to the type
    tol = (3.01 + 2 * k) * 2.0 ** -24 * size
    tol = tol + HALF[dtype] * (exact.abs() + tol) + TINY[dtype]
    assert bool(((got.cpu().double() - exact).abs() <= tol).all())
