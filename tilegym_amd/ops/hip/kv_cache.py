""" "hip" implementations of the operators over the paged e4m3 cache."""

from __future__ import annotations

import torch

from ... import _lib
from ...backend import register_impl


def _one_device(where: str, *tensors) -> None:
    """The kernels take every tensor's address as one of the first tensor's device."""
    device = tensors[0].device
    if device.type != "cuda":
        raise RuntimeError(f"{where}: needs tensors on a HIP device, got one on {device}")
    for t in tensors[1:]:
        if t is not None and t.device != device:
            raise ValueError(f"{where}: tensors on {device} and on {t.device}")


@register_impl("kv_cache_append", backend="hip")
def kv_cache_append(cache, k, v, block_table, seq_lens, indptr, q=None, rope=None, interleaved=False):
    if _lib.native_path():
        done = _lib.native.kv_append(cache, k, v, block_table, seq_lens, indptr, q, rope, interleaved)
        if done is not None:
            return done[0]
    _one_device("kv_cache_append", k, v, *cache, block_table, seq_lens, indptr, q, rope)
    q_out = None
    if q is not None:
        if rope is None:
            raise ValueError("kv_cache_append: q is turned by rope, which is missing")
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    _lib.fp8_kv_append(cache, k, v, block_table, seq_lens, indptr, q_out, q, rope, interleaved)
    return q_out


@register_impl("kv_cache_read", backend="hip")
def kv_cache_read(cache, block_table, indptr, total_tokens, out_dtype=torch.bfloat16, k_out=None, v_out=None):
    if k_out is None and v_out is None and _lib.native_path():
        out = _lib.native.kv_read(cache, block_table, indptr, total_tokens, out_dtype)
        if out is not None:
            return out
    _one_device("kv_cache_read", *cache, block_table, indptr, k_out, v_out)
    if cache[0].dim() != 4:
        raise ValueError("kv_cache_read: the cache's k must be (pages, heads, page size, head dim)")
    shape = (int(total_tokens), cache[0].shape[1], cache[0].shape[3])
    k_out, v_out = (torch.empty(shape, dtype=out_dtype, device=cache[0].device) if t is None else t for t in (k_out, v_out))
    for t in (k_out, v_out):
        if tuple(t.shape) != shape or t.dtype != out_dtype:
            raise ValueError(f"kv_cache_read: k_out and v_out must be {shape} of {out_dtype}, got {tuple(t.shape)} of {t.dtype}")
    _lib.fp8_kv_read(k_out, v_out, cache, block_table, indptr)
    return k_out, v_out


@register_impl("kv_cache_attention", backend="hip")
def kv_cache_attention(q, cache, block_table, seq_lens, indptr, sm_scale=None, window=0, sink_tokens=0, out=None):
    for name, value in (("window", window), ("sink_tokens", sink_tokens)):
        if not 0 <= value < 2 ** 31:
            raise ValueError(f"kv_cache_attention: {name} must be in [0, 2^31), got {value}")
    if sm_scale is None:
        sm_scale = q.shape[-1] ** -0.5 if q.dim() and q.shape[-1] else 1.0
    if _lib.native_path():
        done = _lib.native.kv_attention(q, cache, block_table, seq_lens, indptr, sm_scale, window, sink_tokens, out)
        if done is not None:
            return done
    _one_device("kv_cache_attention", q, *cache, block_table, seq_lens, indptr, out)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    _lib.fp8_kv_attention(out, q, cache, block_table, seq_lens, indptr, sm_scale, window, sink_tokens)
    return out
