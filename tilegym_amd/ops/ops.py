"""Public op stubs with the reference's signatures (src/tilegym/ops/ops.py:715-773).
Bodies only raise; the registered "hip" implementation does the work."""

from __future__ import annotations

from typing import Any, List, Optional, Tuple

import torch

from ..backend import dispatch, get_current_backend


@dispatch("matmul")
def matmul(
    a: torch.Tensor,
    b: torch.Tensor,
    trans_a: Optional[bool] = None,
    trans_b: Optional[bool] = None,
    static_persistent: Optional[bool] = True,
    use_tma: Optional[bool] = None,
    **kwargs: Any,
):
    """Matrix multiplication (src/tilegym/ops/ops.py:715-741).

    a: (M,K), or (K,M) with trans_a;  b: (K,N), or (N,K) with trans_b.  Without extra keywords
    the result has ``a.dtype``, as in the reference (src/tilegym/ops/cutile/matmul.py:446).
    Keyword-only extensions of the "hip" backend for scaled FP8:
      scale_a, scale_b : float | 1-element fp32 tensor (per-tensor) | block scales
                         (M, ceil(K/128)) and (ceil(N/128), ceil(K/128))
      out_dtype        : torch.bfloat16 / float16 / float32
      kernel_configs   : dict of schedule overrides (KERNEL, BLOCK_M, BLOCK_N, SPLIT_K, ROW_GROUPS)
    ``static_persistent`` and ``use_tma`` are accepted and ignored (no such choice on gfx950)."""
    raise NotImplementedError(f"Matmul is not implemented for this backend: {get_current_backend()}")


@dispatch("group_gemm")
def group_gemm(
    group_A: List[torch.Tensor],
    group_B: List[torch.Tensor],
    static_persistent: Optional[bool] = True,
    use_tma: Optional[bool] = True,
    **kwargs: Any,
):
    """List of independent GEMMs (src/tilegym/ops/ops.py:744-773); ``transpose_b`` keyword as in
    src/tilegym/ops/cutile/group_gemm.py:170-197.  "hip" extensions: ``scales_a``/``scales_b``
    (lists, per-tensor or block), ``out_dtype``, ``kernel_configs``."""
    raise NotImplementedError(f"Group GEMM is not implemented for this backend: {get_current_backend()}")


@dispatch("rms_norm_quant")
def rms_norm_quant(
    x: torch.Tensor,
    weight: torch.Tensor,
    eps: float = 1e-6,
    residual: Optional[torch.Tensor] = None,
    group_size: Optional[int] = 128,
    scale: Optional[torch.Tensor] = None,
    residual_out: Optional[torch.Tensor] = None,
    return_norm: bool = False,
) -> Tuple[torch.Tensor, ...]:
    """Root-mean-square norm with the residual's addition and an e4m3 output, in front of an FP8 projection, in one launch
    (in the reference: ``rms_norm``, src/tilegym/ops/ops.py, and a quantizer behind it).

    s = x + residual;  y = s / sqrt(mean(s^2) + eps) * weight;  q = e4m3(y / scale), clamped to +-448, rounded once from the IEEE quotient of
    fp32 y: scales and codes are those of ``act_quant`` on it.
    x (..., H) bf16 / f16 / f32, contiguous, H % 16 == 0, H <= 32768; weight (H), x's type or fp32; residual like x.
    ``scale`` None: 1 x group_size scales amax / 448 as ``act_quant``'s (all-zero group -> 1), H % group_size == 0, group_size 16 /
    32 / 64 / 128: what ``w8a8_block_fp8_matmul`` takes.  Else one fp32 element on the device, for ``matmul(scale_a=scale)``.

    Returns (q, scales), then x + residual rounded to x's type if ``residual`` is given (written to ``residual_out`` if that
    is: it may be ``residual`` or ``x`` itself), then y rounded to x's type if ``return_norm``."""
    raise NotImplementedError(f"rms_norm_quant is not implemented for this backend: {get_current_backend()}")
