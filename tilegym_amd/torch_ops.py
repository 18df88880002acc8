"""The HIP entry points as operators of torch's dispatcher: ``torch.ops.tilegym_hip.*``.

The reference launches its kernels from Python on torch's current stream
(src/tilegym/ops/cutile/matmul.py:446-455); callers that key on torch's dispatcher -- ``torch.compile`` graphs,
``torch.library.opcheck``, anything that enumerates ``torch.ops`` -- cannot see a plain Python function.  Each operator
below is a thin ``torch.library.custom_op`` over the same C-ABI call the ``tilegym_amd.ops`` functions make (one
implementation, two ways in), with a shape-only "fake" implementation so that a graph can be traced without a GPU.
They are registered for device tensors only: with CPU tensors the dispatcher raises (there is no CPU implementation).

    fp8_gemm(a, b, scale_a, scale_b, trans_a, trans_b, alpha, out_dtype) -> c          tg_fp8_gemm
    fp8_gemm_out(c, a, b, scale_a, scale_b, trans_a, trans_b, alpha, beta) -> ()       tg_fp8_gemm, in place
    fp8_ragged_gemm(a, b, a_scale, b_scale, m_indptr, out_dtype) -> c                  tg_fp8_ragged_gemm
    fp8_moe_gemm_out(c, a, b, a_scale, b_scale, topk_weights, sorted_token_ids, expert_ids,
                     num_tokens_post_padded, mul_routed_weight, top_k, block_m) -> ()  tg_fp8_moe_gemm
    fp8_quant_1x128(x) -> (q, scales)                                                   tg_fp8_quant_1x128
    fp8_fused_moe(hidden, w1, w2, w1_scale, w2_scale, topk_weights, topk_ids) -> out   the FP8 MoE layer (tg_fp8_fused_moe
                                                                                        when it fits one chunk)
    fp8_rms_norm_quant(x, weight, eps, residual, group_size, scale, return_norm) -> [q, scales unless scale is given,
                     x + residual if there is one, the norm if asked for]               tg_fp8_rms_norm_quant
    fp8_kv_append(k_cache, v_cache, k_scale, v_scale, k, v, block_table, seq_lens, indptr, rope, interleaved) -> ()
    fp8_kv_append_turn(..., indptr, q, rope, interleaved) -> q turned                   tg_fp8_kv_append; the cache is written in place
    fp8_kv_read(k_cache, v_cache, k_scale, v_scale, block_table, indptr, total_tokens, out_dtype) -> (k, v)    tg_fp8_kv_read
    fp8_kv_attention(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, indptr, sm_scale, window, sink_tokens) -> out
                                                                                        tg_fp8_kv_attention
    int8_gemm(a, b, scale_a, scale_b, bias, out_dtype) -> c                             tg_int8_gemm
    int8_ragged_gemm(a, b, scale_a, scale_b, m_indptr, out_dtype) -> c                  tg_int8_ragged_gemm, rows of no expert zero
    int8_quant(x) -> (q, scales); int8_silu_mul_quant(x) -> (q, scales)                 tg_int8_quant
    int8_permute_quant(x, rows) -> (q, scales)                                          tg_int8_quant, rows carried to their experts
    moe_sort(topk_ids, num_experts) -> (indptr, rows, slots)                            tg_moe_sort
    moe_permute(x, rows) -> out; moe_unpermute(x, rows, weights) -> out                 tg_moe_permute, tg_moe_unpermute; differentiable
    moe_unpermute_backward(grad_out, x, rows, weights) -> (grad_x, grad_weights)        tg_moe_unpermute_backward
What all but the first six take and leave unset is said at ``tilegym_amd.ops``.
"""

from __future__ import annotations

from typing import List, Optional, Tuple

import torch

from . import _lib

NAMESPACE = "tilegym_hip"
OP_NAMES = ("fp8_gemm", "fp8_gemm_out", "fp8_ragged_gemm", "fp8_moe_gemm_out", "fp8_quant_1x128", "fp8_fused_moe", "fp8_rms_norm_quant",
            "fp8_kv_append", "fp8_kv_append_turn", "fp8_kv_read", "fp8_kv_attention", "int8_gemm", "int8_ragged_gemm", "int8_quant", "int8_silu_mul_quant",
            "int8_permute_quant", "moe_sort", "moe_permute", "moe_unpermute", "moe_unpermute_backward")
_CACHE = ("k_cache", "v_cache", "k_scale", "v_scale")


def _mnk(a: torch.Tensor, b: torch.Tensor, trans_a: bool, trans_b: bool) -> Tuple[int, int, int]:
    if a.dim() != 2 or b.dim() != 2:
        raise ValueError("fp8_gemm expects 2-D operands")
    M, K = (a.shape[1], a.shape[0]) if trans_a else (a.shape[0], a.shape[1])
    N, KB = (b.shape[0], b.shape[1]) if trans_b else (b.shape[1], b.shape[0])
    if K != KB:
        raise ValueError(f"Incompatible matrices: K dimension of A is {K}, K dimension of B is {KB}")
    return M, N, K


@torch.library.custom_op(f"{NAMESPACE}::fp8_gemm", mutates_args=(), device_types="cuda")
def fp8_gemm(a: torch.Tensor, b: torch.Tensor, scale_a: Optional[torch.Tensor], scale_b: Optional[torch.Tensor],
             trans_a: bool, trans_b: bool, alpha: float, out_dtype: torch.dtype) -> torch.Tensor:
    M, N, _ = _mnk(a, b, trans_a, trans_b)
    c = torch.empty((M, N), dtype=out_dtype, device=a.device)
    _lib.fp8_gemm(c, a, b, scale_a, scale_b, trans_a, trans_b, alpha, 0.0)
    return c


@fp8_gemm.register_fake
def _(a, b, scale_a, scale_b, trans_a, trans_b, alpha, out_dtype):
    M, N, _ = _mnk(a, b, trans_a, trans_b)
    return a.new_empty((M, N), dtype=out_dtype)


@torch.library.custom_op(f"{NAMESPACE}::fp8_gemm_out", mutates_args=("c",), device_types="cuda")
def fp8_gemm_out(c: torch.Tensor, a: torch.Tensor, b: torch.Tensor, scale_a: Optional[torch.Tensor],
                 scale_b: Optional[torch.Tensor], trans_a: bool, trans_b: bool, alpha: float, beta: float) -> None:
    _lib.fp8_gemm(c, a, b, scale_a, scale_b, trans_a, trans_b, alpha, beta)


@fp8_gemm_out.register_fake
def _(c, a, b, scale_a, scale_b, trans_a, trans_b, alpha, beta):
    M, N, _ = _mnk(a, b, trans_a, trans_b)
    if tuple(c.shape) != (M, N):
        raise ValueError(f"c must be ({M}, {N})")


@torch.library.custom_op(f"{NAMESPACE}::fp8_ragged_gemm", mutates_args=(), device_types="cuda")
def fp8_ragged_gemm(a: torch.Tensor, b: torch.Tensor, a_scale: Optional[torch.Tensor], b_scale: torch.Tensor,
                    m_indptr: torch.Tensor, out_dtype: torch.dtype) -> torch.Tensor:
    # rows past m_indptr[-1] belong to no expert and are not written: they read as zero
    c = torch.zeros((a.shape[0], b.shape[1]), dtype=out_dtype, device=a.device)
    _lib.fp8_ragged_gemm(c, a, b, a_scale, b_scale, m_indptr)
    return c


@fp8_ragged_gemm.register_fake
def _(a, b, a_scale, b_scale, m_indptr, out_dtype):
    if a.dim() != 2 or b.dim() != 3 or a.shape[1] != b.shape[2]:
        raise ValueError("fp8_ragged_gemm expects a (rows, K) and b (experts, N, K)")
    return a.new_empty((a.shape[0], b.shape[1]), dtype=out_dtype)


@torch.library.custom_op(f"{NAMESPACE}::fp8_moe_gemm_out", mutates_args=("c",), device_types="cuda")
def fp8_moe_gemm_out(c: torch.Tensor, a: torch.Tensor, b: torch.Tensor, a_scale: Optional[torch.Tensor],
                     b_scale: Optional[torch.Tensor], topk_weights: Optional[torch.Tensor], sorted_token_ids: torch.Tensor,
                     expert_ids: torch.Tensor, num_tokens_post_padded: torch.Tensor, mul_routed_weight: bool, top_k: int,
                     block_m: int) -> None:
    _lib.fp8_moe_gemm(c.view(-1, c.shape[-1]), a, b, a_scale, b_scale, topk_weights, sorted_token_ids, expert_ids,
                      num_tokens_post_padded, mul_routed_weight, top_k, block_m)


@fp8_moe_gemm_out.register_fake
def _(c, a, b, a_scale, b_scale, topk_weights, sorted_token_ids, expert_ids, num_tokens_post_padded, mul_routed_weight,
      top_k, block_m):
    if b.dim() != 3 or a.shape[-1] != b.shape[2] or c.shape[-1] != b.shape[1]:
        raise ValueError("fp8_moe_gemm_out expects a (tokens, K), b (experts, N, K) and c (..., N)")


@torch.library.custom_op(f"{NAMESPACE}::fp8_quant_1x128", mutates_args=(), device_types="cuda")
def fp8_quant_1x128(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    q, scales = _lib.fp8_quant_1x128(x.contiguous(), 0.0, False)
    return q, scales


@fp8_quant_1x128.register_fake
def _(x):
    if x.shape[-1] % 128 != 0:
        raise ValueError("the last dimension must be a multiple of 128")
    return x.new_empty(x.shape, dtype=torch.float8_e4m3fn), x.new_empty(x.shape[:-1] + (x.shape[-1] // 128,), dtype=torch.float32)


@torch.library.custom_op(f"{NAMESPACE}::fp8_fused_moe", mutates_args=(), device_types="cuda")
def fp8_fused_moe(hidden: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor, w1_scale: torch.Tensor, w2_scale: torch.Tensor,
                  topk_weights: torch.Tensor, topk_ids: torch.Tensor) -> torch.Tensor:
    from .ops.moe_interface import fused_experts_impl
    return fused_experts_impl(hidden, w1, w2, topk_weights, topk_ids, inplace=False, use_fp8_w8a8=True, w1_scale=w1_scale,
                              w2_scale=w2_scale)


@fp8_fused_moe.register_fake
def _(hidden, w1, w2, w1_scale, w2_scale, topk_weights, topk_ids):
    if hidden.dim() != 2 or w1.dim() != 3 or w2.dim() != 3 or w1.shape[2] != hidden.shape[1] or w2.shape[1] != hidden.shape[1]:
        raise ValueError("fp8_fused_moe expects hidden (T, H), w1 (E, 2I, H) and w2 (E, H, I)")
    return hidden.new_empty(hidden.shape, dtype=torch.bfloat16 if hidden.dtype == torch.bfloat16 else torch.float16)


@torch.library.custom_op(f"{NAMESPACE}::fp8_rms_norm_quant", mutates_args=(), device_types="cuda")
def fp8_rms_norm_quant(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: Optional[torch.Tensor], group_size: int,
                       scale: Optional[torch.Tensor], return_norm: bool) -> List[torch.Tensor]:
    from .ops import rms_norm_quant
    q, scales, *rest = rms_norm_quant(x, weight, eps, residual=residual, group_size=group_size, scale=scale, return_norm=return_norm)
    return [q, *rest] if scale is not None else [q, scales, *rest]  # (an operator's results are no inputs of it)


@fp8_rms_norm_quant.register_fake
def _(x, weight, eps, residual, group_size, scale, return_norm):
    out = [x.new_empty(x.shape, dtype=torch.float8_e4m3fn)]
    if scale is None:
        if group_size not in (16, 32, 64, 128) or x.shape[-1] % group_size != 0:
            raise ValueError(f"fp8_rms_norm_quant: rows of {x.shape[-1]} in groups of {group_size}")
        out.append(x.new_empty(x.shape[:-1] + (x.shape[-1] // group_size,), dtype=torch.float32))
    return out + [x.new_empty(x.shape) for wanted in (residual is not None, return_norm) if wanted]


def _cache_of(k_cache, v_cache, k_scale, v_scale):
    from .ops import KVCache
    return KVCache(k_cache, v_cache, k_scale, v_scale)


def _check_heads(k_cache: torch.Tensor, x: torch.Tensor, name: str) -> None:
    if k_cache.dim() != 4 or x.dim() != 3 or x.shape[2] != k_cache.shape[3]:
        raise ValueError(f"{name} expects a cache (pages, heads, page size, D) and packed (tokens, heads, D)")


@torch.library.custom_op(f"{NAMESPACE}::fp8_kv_append", mutates_args=_CACHE, device_types="cuda")
def fp8_kv_append(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                  block_table: torch.Tensor, seq_lens: torch.Tensor, indptr: torch.Tensor, rope: Optional[torch.Tensor], interleaved: bool) -> None:
    from .ops import kv_cache_append
    kv_cache_append(_cache_of(k_cache, v_cache, k_scale, v_scale), k, v, block_table, seq_lens, indptr, rope=rope, interleaved=interleaved)


@fp8_kv_append.register_fake
def _(k_cache, v_cache, k_scale, v_scale, k, v, block_table, seq_lens, indptr, rope, interleaved):
    _check_heads(k_cache, k, "fp8_kv_append")


@torch.library.custom_op(f"{NAMESPACE}::fp8_kv_append_turn", mutates_args=_CACHE, device_types="cuda")
def fp8_kv_append_turn(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                       block_table: torch.Tensor, seq_lens: torch.Tensor, indptr: torch.Tensor, q: torch.Tensor, rope: torch.Tensor,
                       interleaved: bool) -> torch.Tensor:
    from .ops import kv_cache_append
    return kv_cache_append(_cache_of(k_cache, v_cache, k_scale, v_scale), k, v, block_table, seq_lens, indptr, q=q, rope=rope, interleaved=interleaved)


@fp8_kv_append_turn.register_fake
def _(k_cache, v_cache, k_scale, v_scale, k, v, block_table, seq_lens, indptr, q, rope, interleaved):
    _check_heads(k_cache, k, "fp8_kv_append_turn"), _check_heads(k_cache, q, "fp8_kv_append_turn")
    return q.new_empty(q.shape)


@torch.library.custom_op(f"{NAMESPACE}::fp8_kv_read", mutates_args=(), device_types="cuda")
def fp8_kv_read(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, block_table: torch.Tensor, indptr: torch.Tensor,
                total_tokens: int, out_dtype: torch.dtype) -> Tuple[torch.Tensor, torch.Tensor]:
    from .ops import kv_cache_read
    return kv_cache_read(_cache_of(k_cache, v_cache, k_scale, v_scale), block_table, indptr, total_tokens, out_dtype)


@fp8_kv_read.register_fake
def _(k_cache, v_cache, k_scale, v_scale, block_table, indptr, total_tokens, out_dtype):
    if k_cache.dim() != 4:
        raise ValueError("fp8_kv_read expects a cache (pages, heads, page size, D)")
    shape = (total_tokens, k_cache.shape[1], k_cache.shape[3])
    return k_cache.new_empty(shape, dtype=out_dtype), k_cache.new_empty(shape, dtype=out_dtype)


@torch.library.custom_op(f"{NAMESPACE}::fp8_kv_attention", mutates_args=(), device_types="cuda")
def fp8_kv_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, block_table: torch.Tensor,
                     seq_lens: torch.Tensor, indptr: torch.Tensor, sm_scale: Optional[float], window: int, sink_tokens: int) -> torch.Tensor:
    from .ops import kv_cache_attention
    return kv_cache_attention(q, _cache_of(k_cache, v_cache, k_scale, v_scale), block_table, seq_lens, indptr, sm_scale=sm_scale, window=window,
                              sink_tokens=sink_tokens)


@fp8_kv_attention.register_fake
def _(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, indptr, sm_scale, window, sink_tokens):
    _check_heads(k_cache, q, "fp8_kv_attention")
    return q.new_empty(q.shape)


@torch.library.custom_op(f"{NAMESPACE}::int8_gemm", mutates_args=(), device_types="cuda")
def int8_gemm(a: torch.Tensor, b: torch.Tensor, scale_a: torch.Tensor, scale_b: torch.Tensor, bias: Optional[torch.Tensor], out_dtype: torch.dtype) -> torch.Tensor:
    from .ops import int8_matmul
    return int8_matmul(a, b, scale_a, scale_b, bias=bias, out_dtype=out_dtype)


@int8_gemm.register_fake
def _(a, b, scale_a, scale_b, bias, out_dtype):
    if a.dim() < 1 or b.dim() != 2 or a.shape[-1] != b.shape[1]:
        raise ValueError("int8_gemm expects a (..., K) and b (N, K)")
    return a.new_empty(a.shape[:-1] + b.shape[:1], dtype=out_dtype)


@torch.library.custom_op(f"{NAMESPACE}::int8_ragged_gemm", mutates_args=(), device_types="cuda")
def int8_ragged_gemm(a: torch.Tensor, b: torch.Tensor, scale_a: torch.Tensor, scale_b: torch.Tensor, m_indptr: torch.Tensor,
                     out_dtype: torch.dtype) -> torch.Tensor:
    from .ops import ragged_int8_matmul
    out = torch.zeros((a.shape[0], b.shape[1]), dtype=out_dtype, device=a.device)
    return ragged_int8_matmul(a, b, scale_a, scale_b, m_indptr, out_dtype=out_dtype, out=out)


@int8_ragged_gemm.register_fake
def _(a, b, scale_a, scale_b, m_indptr, out_dtype):
    if a.dim() != 2 or b.dim() != 3 or a.shape[1] != b.shape[2]:
        raise ValueError("int8_ragged_gemm expects a (rows, K) and b (experts, N, K)")
    return a.new_empty((a.shape[0], b.shape[1]), dtype=out_dtype)


@torch.library.custom_op(f"{NAMESPACE}::int8_quant", mutates_args=(), device_types="cuda")
def int8_quant(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    from .ops import quant_int8
    return quant_int8(x)


@int8_quant.register_fake
def _(x):
    return x.new_empty(x.shape, dtype=torch.int8), x.new_empty(x.shape[:-1], dtype=torch.float32)


@torch.library.custom_op(f"{NAMESPACE}::int8_silu_mul_quant", mutates_args=(), device_types="cuda")
def int8_silu_mul_quant(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    from .ops import silu_mul_quant_int8
    return silu_mul_quant_int8(x)


@int8_silu_mul_quant.register_fake
def _(x):
    if x.shape[-1] % 2 != 0:
        raise ValueError("int8_silu_mul_quant expects x (..., 2 I)")
    return x.new_empty(x.shape[:-1] + (x.shape[-1] // 2,), dtype=torch.int8), x.new_empty(x.shape[:-1], dtype=torch.float32)


def _order_of(rows):
    """The operators over a MoeOrder read its rows only."""
    from .ops import MoeOrder
    return MoeOrder(rows, rows, rows)


def _check_rows(name: str, x: torch.Tensor, rows: torch.Tensor, n) -> None:
    if x.dim() != 2 or rows.dim() != 2 or x.shape[0] != n:
        raise ValueError(f"{name}: x {tuple(x.shape)} does not go with rows {tuple(rows.shape)}")


@torch.library.custom_op(f"{NAMESPACE}::int8_permute_quant", mutates_args=(), device_types="cuda")
def int8_permute_quant(x: torch.Tensor, rows: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    from .ops import moe_permute_quant_int8
    return moe_permute_quant_int8(x, _order_of(rows))


@int8_permute_quant.register_fake
def _(x, rows):
    _check_rows("int8_permute_quant", x, rows, rows.shape[0])
    return x.new_empty((rows.numel(), x.shape[1]), dtype=torch.int8), x.new_empty((rows.numel(),), dtype=torch.float32)


@torch.library.custom_op(f"{NAMESPACE}::moe_sort", mutates_args=(), device_types="cuda")
def moe_sort(topk_ids: torch.Tensor, num_experts: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    from .ops import moe_sort as sort
    return tuple(sort(topk_ids, num_experts))


@moe_sort.register_fake
def _(topk_ids, num_experts):
    i32 = dict(dtype=torch.int32)
    return topk_ids.new_empty((num_experts + 1,), **i32), topk_ids.new_empty(topk_ids.shape, **i32), topk_ids.new_empty((topk_ids.numel(),), **i32)


@torch.library.custom_op(f"{NAMESPACE}::moe_permute", mutates_args=(), device_types="cuda")
def moe_permute(x: torch.Tensor, rows: torch.Tensor) -> torch.Tensor:
    from .ops import moe_permute as permute
    return permute(x, _order_of(rows))


@moe_permute.register_fake
def _(x, rows):
    _check_rows("moe_permute", x, rows, rows.shape[0])
    return x.new_empty((rows.numel(), x.shape[1]))


@torch.library.custom_op(f"{NAMESPACE}::moe_unpermute", mutates_args=(), device_types="cuda")
def moe_unpermute(x: torch.Tensor, rows: torch.Tensor, weights: Optional[torch.Tensor]) -> torch.Tensor:
    from .ops import moe_unpermute as unpermute
    return unpermute(x, _order_of(rows), weights)


@moe_unpermute.register_fake
def _(x, rows, weights):
    _check_rows("moe_unpermute", x, rows, rows.numel())
    return x.new_empty((rows.shape[0], x.shape[1]))


@torch.library.custom_op(f"{NAMESPACE}::moe_unpermute_backward", mutates_args=(), device_types="cuda")
def moe_unpermute_backward(grad_out: torch.Tensor, x: torch.Tensor, rows: torch.Tensor, weights: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    from .ops import moe_unpermute_backward as backward
    return backward(grad_out, x, _order_of(rows), weights)


@moe_unpermute_backward.register_fake
def _(grad_out, x, rows, weights):
    _check_rows("moe_unpermute_backward", x, rows, rows.numel())
    return x.new_empty(x.shape), weights.new_empty(weights.shape)


def _recordable(name: str, *leaves) -> None:
    """The operators themselves run below autograd and see no gradients: what they refuse of a capture is looked for where a graph is recorded."""
    from .ops.hip.moe_route import _recordable as check
    check(name, *leaves)


def _save_permute(ctx, inputs, output):
    _recordable("moe_permute", inputs[0])
    ctx.save_for_backward(inputs[1])


def _save_unpermute(ctx, inputs, output):
    x, rows, weights = inputs
    _recordable("moe_unpermute", x, weights)
    ctx.weighted = weights is not None
    ctx.save_for_backward(rows, *([x, weights] if ctx.weighted else []))


def _grad_permute(ctx, grad):
    return torch.ops.tilegym_hip.moe_unpermute(grad.contiguous(), ctx.saved_tensors[0], None), None


def _grad_unpermute(ctx, grad):
    rows = ctx.saved_tensors[0]
    if not ctx.weighted:
        return torch.ops.tilegym_hip.moe_permute(grad.contiguous(), rows), None, None
    grad_x, grad_weights = torch.ops.tilegym_hip.moe_unpermute_backward(grad, ctx.saved_tensors[1], rows, ctx.saved_tensors[2])
    return grad_x, None, grad_weights


moe_permute.register_autograd(_grad_permute, setup_context=_save_permute)
moe_unpermute.register_autograd(_grad_unpermute, setup_context=_save_unpermute)


def registered_ops():
    """Names of the operators this module registered, as ``torch.ops`` sees them."""
    ns = getattr(torch.ops, NAMESPACE)
    return [f"{NAMESPACE}::{name}" for name in OP_NAMES if hasattr(ns, name)]
