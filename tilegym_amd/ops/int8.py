"""Products in 8-bit integers with a scale per token and per output channel, and the quantizers in front of them.  None of them has a gradient.

The reference's counterparts are the int8 forms of its MoE interface (``use_int8_w8a16``, src/tilegym/ops/moe_interface.py:116-322) and
``per_token_group_quant_8bit`` (src/tilegym/suites/flashinfer/ops.py), whose int8 codes no product of it takes."""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from ..backend import dispatch, get_current_backend


@dispatch("int8_matmul")
def int8_matmul(
    a: torch.Tensor,
    b: torch.Tensor,
    scale_a: torch.Tensor,
    scale_b: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    out_dtype: torch.dtype = torch.bfloat16,
    out: Optional[torch.Tensor] = None,
    kernel_configs: Optional[dict] = None,
) -> torch.Tensor:
    """out[..., n] = scale_a[...] * scale_b[n] * sum_k a[..., k] * b[n, k] + bias[n], in one launch, or two where K is split.

    a (..., K) and b (N, K) int8, contiguous; scale_a fp32 with one element per row of a, or one for all; scale_b fp32 with N elements, or
    one; bias (N) bf16 / f16 / fp32.  The sums are exact (32-bit integers, K at most 131071); the scales and the bias are applied in fp32 and the
    result is rounded once to ``out_dtype`` (bf16 / f16 / fp32).  The bits do not depend on the number of rows, the kernel or the split.

    Any sizes are taken; rows whose length is a multiple of 16 bytes, at 16-byte addresses, by the fast kernels.  ``out`` (contiguous, ``out_dtype``)
    is written if given.  ``kernel_configs``: KERNEL, BLOCK_M, BLOCK_N, SPLIT_K as for ``matmul``."""
    raise NotImplementedError(f"int8_matmul is not implemented for this backend: {get_current_backend()}")


@dispatch("ragged_int8_matmul")
def ragged_int8_matmul(
    a: torch.Tensor,
    b: torch.Tensor,
    scale_a: torch.Tensor,
    scale_b: torch.Tensor,
    m_indptr: torch.Tensor,
    out_dtype: torch.dtype = torch.bfloat16,
    out: Optional[torch.Tensor] = None,
    kernel_configs: Optional[dict] = None,
) -> torch.Tensor:
    """``int8_matmul`` of each expert's rows with its weight: rows m_indptr[e] : m_indptr[e + 1] of a (M, K) with b[e] of b (E, N, K) and scale_b[e]
    of scale_b (E, N).  scale_a has M elements, or one; scale_b E * N, or one.  ``m_indptr`` (E + 1) int32 on the device, non-decreasing, is not read by
    the host (``MoeOrder.indptr``); M is below 2^29.  Rows of no expert are left as they were in ``out``, and unset without it."""
    raise NotImplementedError(f"ragged_int8_matmul is not implemented for this backend: {get_current_backend()}")


@dispatch("quant_int8")
def quant_int8(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """A scale per row and its codes: (q, scales), q int8 like x (..., K), scales fp32 (...).

    scale = max|x| * fp32(1 / 127) (1 for a row of zeros, and for one so small that this product is zero), q = x / scale, an IEEE quotient in
    fp32, rounded half to even, within +-127.  A row that holds a NaN or an infinity gets the scale NaN and codes of zero.  x bf16 / f16 /
    fp32, contiguous.  A weight (N, K) becomes b and scale_b of ``int8_matmul`` in the same way."""
    raise NotImplementedError(f"quant_int8 is not implemented for this backend: {get_current_backend()}")


@dispatch("silu_mul_quant_int8")
def silu_mul_quant_int8(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``quant_int8`` of silu(x[..., :I]) * x[..., I:] for x (..., 2 I): what lies between a gated layer's two products, in one launch.  The
    activation is fp32 and is not rounded before it is quantized."""
    raise NotImplementedError(f"silu_mul_quant_int8 is not implemented for this backend: {get_current_backend()}")


def int8_moe(
    hidden_states: torch.Tensor,
    w1: torch.Tensor,
    w2: torch.Tensor,
    w1_scale: torch.Tensor,
    w2_scale: torch.Tensor,
    topk_weights: torch.Tensor,
    topk_ids: torch.Tensor,
    rows_dtype: Optional[torch.dtype] = None,
) -> torch.Tensor:
    """A gated layer of experts in int8: sort -> permute and quantize -> gate and up -> SiLU(gate) * up, quantized -> down -> back, weighted.

    hidden_states (T, H) bf16 / f16; w1 (E, 2 I, H), w2 (E, H, I) int8 with scales per output channel w1_scale (E, 2 I), w2_scale (E, H) fp32;
    topk_weights (T, k) fp32 / bf16 / f16; topk_ids (T, k) int32 / int64.  A slot whose id is outside [0, E) (an expert of another rank, say) adds
    nothing.  Returns (T, H), without a gradient, in the weights either.

    Both products' outputs are rounded to hidden_states' type, the second one's before they are weighted and summed (in fp32) and rounded again: half the bytes to write and
    to gather, for one more rounding of each row.  ``rows_dtype=torch.float32`` keeps the second product's rows whole, and the sum is all that is rounded
    behind it (bf16, 64 experts of inter 1408, rows of 2048: error against 64 bits 0.0025 -> 0.0019; 4096 tokens 361 -> 402 us, 8 tokens 65 -> 67)."""
    from .. import _lib
    from .moe_route import moe_permute_quant_int8, moe_sort, moe_unpermute

    if rows_dtype not in (None, hidden_states.dtype, torch.float32):
        raise ValueError(f"int8_moe: rows_dtype must be {hidden_states.dtype} or torch.float32, got {rows_dtype}")
    whole = rows_dtype is torch.float32
    if not whole and _lib.native_path():  # the six launches below in one call
        out = _lib.native.int8_moe(hidden_states, w1, w2, w1_scale, w2_scale, topk_weights, topk_ids)
        if out is not None:
            return out
    if hidden_states.dtype not in (torch.bfloat16, torch.float16):
        raise NotImplementedError(f"int8_moe: hidden_states must be bf16 or f16, got {hidden_states.dtype}")
    order = moe_sort(topk_ids, w1.shape[0])
    q, scales = moe_permute_quant_int8(hidden_states, order)
    h = ragged_int8_matmul(q, w1, scales, w1_scale, order.indptr, out_dtype=hidden_states.dtype)
    q, scales = silu_mul_quant_int8(h)
    y = ragged_int8_matmul(q, w2, scales, w2_scale, order.indptr, out_dtype=torch.float32 if whole else hidden_states.dtype)
    return moe_unpermute(y, order, topk_weights.detach()).to(hidden_states.dtype)
