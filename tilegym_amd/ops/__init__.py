"""tilegym.ops-shaped namespace: public stubs + the "hip" implementations (registered on import)."""

from . import hip  # noqa: F401  (registers implementations)
from .kv_cache import KVCache, alloc_kv_cache, kv_cache_append, kv_cache_attention, kv_cache_read, rope_table
from .moe_interface import fused_experts_impl, fused_moe, invoke_fused_moe_kernel, moe_align_block_size
from .ops import group_gemm, matmul, rms_norm_quant

__all__ = ["matmul", "group_gemm", "fused_moe", "fused_experts_impl", "invoke_fused_moe_kernel", "moe_align_block_size",
           "rms_norm_quant", "KVCache", "alloc_kv_cache", "rope_table", "kv_cache_append", "kv_cache_read", "kv_cache_attention"]
