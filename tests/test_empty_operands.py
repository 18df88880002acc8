"""Tensors without elements at the C ABI: the FP8 entry points take none whose strides are not those of their shape (a product over no K, rows of no elements), the int8
and routing operators take them whatever their strides."""

import torch

from tilegym_amd import _lib

from .test_int8_ops import BF16

FP8 = torch.float8_e4m3fn


def test_fp8_entry_points_refuse_lengths_of_zero():
    d, L, (cfg, n) = _lib._desc, _lib.load(), _lib.make_cfg(None)
    a, b, c, one = torch.zeros(5, 0, dtype=torch.uint8).view(FP8), torch.zeros(7, 0, dtype=torch.uint8).view(FP8), torch.zeros(5, 7, dtype=BF16), torch.ones(1)
    b3 = torch.zeros(2, 7, 0, dtype=torch.uint8).view(FP8)
    indptr = torch.tensor([0, 2, 5], dtype=torch.int32)
    x, codes, scales = torch.zeros(5, 0, dtype=BF16), torch.zeros(5, 0, dtype=torch.uint8).view(FP8), torch.zeros(5, 0)

    def error():
        return L.tg_last_error().decode()

    assert L.tg_fp8_gemm(d(c), d(a), d(b), d(one), d(one), 0, 1, 1.0, 0.0, None, cfg, n, 9999, 0) == -6 and "contiguous" in error()
    assert L.tg_fp8_ragged_gemm(d(c), d(a), d(b3), d(one), d(one), d(indptr), cfg, n, 9999, 0) == -6 and "contiguous" in error()
    assert L.tg_fp8_quant_1x128(d(codes), d(scales), d(x), 1e-10, 0, 9999, 0) == -6 and "contiguous" in error()
    assert L.tg_moe_sum(d(torch.zeros(5, 0, dtype=BF16)), d(torch.zeros(5, 2, 0, dtype=BF16)), 9999, 0) == -6 and "contiguous" in error()


def test_int8_and_routing_take_tensors_without_elements():
    d, L, i32 = _lib._desc, _lib.load(), torch.int32
    none = torch.zeros(4, 0, dtype=torch.int8)
    assert L.tg_moe_permute(d(torch.zeros(6, 0)), d(torch.zeros(3, 0)), d(torch.zeros(3, 2, dtype=i32)), 9999, 0) == 0
    assert L.tg_moe_unpermute(d(torch.zeros(3, 0)), d(torch.zeros(1, 1).expand(6, 0)), d(torch.zeros(3, 2, dtype=i32)), None, 9999, 0) == 0
    cfg, n = _lib.make_cfg(None)
    # (a sum over nothing is none of the products, and says so)
    rc = L.tg_int8_gemm(d(torch.zeros(4, 8, dtype=BF16)), d(none), d(torch.zeros(8, 0, dtype=torch.int8)), d(torch.ones(1)), d(torch.ones(1)), None, None, cfg, n, 9999, 0)
    assert rc == -6 and "K must be" in L.tg_last_error().decode()
