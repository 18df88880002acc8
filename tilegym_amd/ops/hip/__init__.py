"""Implementations registered under backend "hip" (one per public op)."""

from . import gemm, int8, kv_cache, moe, moe_route  # noqa: F401
from ... import quant  # noqa: F401  (registers rms_norm_quant)
