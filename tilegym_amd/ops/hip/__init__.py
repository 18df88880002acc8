"""Implementations registered under backend "hip" (one per public op)."""

from . import gemm, kv_cache, moe  # noqa: F401
from ... import quant  # noqa: F401  (registers rms_norm_quant)
