""" "hip" implementations of the products in 8-bit integers and their quantizers."""

from __future__ import annotations

import torch

from ... import _lib
from ...backend import register_impl
from .kv_cache import _one_device


def _output(where, out, shape, dtype, device):
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device)
    if tuple(out.shape) != tuple(shape) or out.dtype != dtype:
        raise ValueError(f"{where}: out must be {tuple(shape)} of {dtype}, got {tuple(out.shape)} of {out.dtype}")
    return out


@register_impl("int8_matmul", backend="hip")
def int8_matmul(a, b, scale_a, scale_b, bias=None, out_dtype=torch.bfloat16, out=None, kernel_configs=None):
    if kernel_configs is None and _lib.native_path():
        c = _lib.native.int8_matmul(a, b, scale_a, scale_b, bias, out_dtype, out)
        if c is not None:
            return c
    _one_device("int8_matmul", a, b, scale_a, scale_b, bias, out)
    if a.dim() < 1 or b.dim() != 2:
        raise ValueError(f"int8_matmul: a must be (..., K) and b (N, K), got {tuple(a.shape)} and {tuple(b.shape)}")
    if not a.is_contiguous():
        raise ValueError("int8_matmul: a must be contiguous")
    out = _output("int8_matmul", out, a.shape[:-1] + b.shape[:1], out_dtype, a.device)
    if not out.is_contiguous():
        raise ValueError("int8_matmul: out must be contiguous")
    rows = 1
    for n in a.shape[:-1]:
        rows *= n
    _lib.int8_gemm(out.view(rows, b.shape[0]), a.view(rows, a.shape[-1]), b, scale_a, scale_b, bias, kernel_configs)
    return out


@register_impl("ragged_int8_matmul", backend="hip")
def ragged_int8_matmul(a, b, scale_a, scale_b, m_indptr, out_dtype=torch.bfloat16, out=None, kernel_configs=None):
    if kernel_configs is None and _lib.native_path():
        c = _lib.native.ragged_int8_matmul(a, b, scale_a, scale_b, m_indptr, out_dtype, out)
        if c is not None:
            return c
    _one_device("ragged_int8_matmul", a, b, scale_a, scale_b, m_indptr, out)
    if a.dim() != 2 or b.dim() != 3:
        raise ValueError(f"ragged_int8_matmul: a must be (M, K) and b (E, N, K), got {tuple(a.shape)} and {tuple(b.shape)}")
    out = _output("ragged_int8_matmul", out, (a.shape[0], b.shape[1]), out_dtype, a.device)
    _lib.int8_ragged_gemm(out, a, b, scale_a, scale_b, m_indptr, kernel_configs)
    return out


@register_impl("quant_int8", backend="hip")
def quant_int8(x):
    if _lib.native_path():
        done = _lib.native.int8_quant(x, None, False)
        if done is not None:
            return done
    _one_device("quant_int8", x)
    if x.dim() < 1:
        raise ValueError("quant_int8: x needs at least one dimension")
    q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scales = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    _lib.int8_quant(q, scales, x)
    return q, scales


@register_impl("silu_mul_quant_int8", backend="hip")
def silu_mul_quant_int8(x):
    if _lib.native_path():
        done = _lib.native.int8_quant(x, None, True)
        if done is not None:
            return done
    _one_device("silu_mul_quant_int8", x)
    if x.dim() < 1 or x.shape[-1] % 2 != 0:
        raise ValueError(f"silu_mul_quant_int8: x must be (..., 2 I), got {tuple(x.shape)}")
    q = torch.empty(x.shape[:-1] + (x.shape[-1] // 2,), dtype=torch.int8, device=x.device)
    scales = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    _lib.int8_quant(q, scales, x, silu_mul=True)
    return q, scales
