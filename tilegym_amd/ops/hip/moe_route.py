""" "hip" implementations of sorting tokens by expert, of the ways there and back, and of their gradients."""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from ... import _lib
from ...backend import register_impl
from ..moe_route import MoeOrder
from .kv_cache import _one_device


def _pairs(where, order):
    rows = order.rows
    if rows.dim() != 2:
        raise ValueError(f"{where}: the order's rows must be (T, k), got {tuple(rows.shape)}")
    return rows.shape[0], rows.shape[1]


def _without_tangents(where, *inputs):
    """A dual tensor need not require a gradient: without a look at it the result would come back without its tangent.  (The native calls leave these to here.)"""
    for t in inputs:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{where}: there are no forward-mode derivatives; only reverse mode is implemented")


def _permute(x, order):
    if _lib.native_path():
        done = _lib.native.moe_permute(x, order.rows)
        if done is not None:
            return done
    _without_tangents("moe_permute", x)
    _one_device("moe_permute", x, order.rows)
    tokens, k = _pairs("moe_permute", order)
    if x.dim() != 2 or x.shape[0] != tokens:
        raise ValueError(f"moe_permute: x must have a row for each of {tokens} tokens, got {tuple(x.shape)}")
    out = torch.empty((tokens * k, x.shape[1]), dtype=x.dtype, device=x.device)
    _lib.moe_permute(out, x, order.rows)
    return out


def _unpermute(x, order, weights, where="moe_unpermute"):
    if _lib.native_path():
        done = _lib.native.moe_unpermute(x, order.rows, weights)
        if done is not None:
            return done
    _without_tangents(where, x, weights)
    _one_device(where, x, order.rows, weights)
    tokens, k = _pairs(where, order)
    if x.dim() != 2 or x.shape[0] != tokens * k:
        raise ValueError(f"{where}: x must have {tokens * k} rows, got {tuple(x.shape)}")
    out = torch.empty((tokens, x.shape[1]), dtype=x.dtype, device=x.device)
    _lib.moe_unpermute(out, x, order.rows, weights)
    return out


def _recordable(where, *leaves):
    """Under capture a leaf's gradient is added to on the stream of the graph that first used it.  Where that is an eager graph which still lives, the backward
    pass would wait for its stream from within the capture, an error that torch's backward threads do not survive: refused here instead."""
    if not torch.cuda.is_initialized() or not torch.cuda.is_current_stream_capturing():  # (shapes may be inferred where there is no device to ask)
        return
    for t in leaves:
        if t is not None and t.requires_grad and t.is_leaf and (not _lib.native_path() or _lib.native.leaf_held(t)):
            raise RuntimeError(f"{where}: an eager graph of this leaf is alive on another stream; release what it computed (its loss, its outputs) before "
                               f"the leaf's forward and backward passes are captured" if _lib.native_path() else
                               f"{where}: without tilegym_amd/_native.so no graph is captured whose leaves take gradients")


class _Permute(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, indptr, rows, slots):
        order = MoeOrder(indptr, rows, slots)
        ctx.save_for_backward(*order)
        return _permute(x, order)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        return _unpermute(grad.contiguous(), MoeOrder(*ctx.saved_tensors), None, "moe_permute_backward"), None, None, None


class _Unpermute(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weights, indptr, rows, slots):
        order = MoeOrder(indptr, rows, slots)
        ctx.save_for_backward(*([x, weights] if weights is not None else []), *order)
        ctx.weighted = weights is not None
        return _unpermute(x, order, weights)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        if not ctx.weighted:
            return _permute(grad.contiguous(), MoeOrder(*ctx.saved_tensors)), None, None, None, None
        x, weights, *order = ctx.saved_tensors
        return (*moe_unpermute_backward(grad, x, MoeOrder(*order), weights), None, None, None)


@register_impl("moe_sort", backend="hip")
def moe_sort(topk_ids, num_experts):
    if _lib.native_path():
        done = _lib.native.moe_sort(topk_ids, num_experts)
        if done is not None:
            return MoeOrder(*done)
    _one_device("moe_sort", topk_ids)
    if topk_ids.dim() != 2:
        raise ValueError(f"moe_sort: topk_ids must be (T, k), got {tuple(topk_ids.shape)}")
    i32 = dict(dtype=torch.int32, device=topk_ids.device)
    order = MoeOrder(torch.empty(min(max(int(num_experts), 0), 512) + 1, **i32), torch.empty(topk_ids.shape, **i32), torch.empty(topk_ids.numel(), **i32))
    _lib.moe_sort(topk_ids.contiguous(), num_experts, *order)
    return order


@register_impl("moe_permute", backend="hip")
def moe_permute(x, order):
    if torch.is_grad_enabled() and x.requires_grad:
        _without_tangents("moe_permute", x)
        _recordable("moe_permute", x)
        if _lib.native_path():
            done = _lib.native.moe_permute_grad(x, order.rows)
            if done is not None:
                return done
        return _Permute.apply(x, *order)
    return _permute(x, order)


@register_impl("moe_permute_quant_int8", backend="hip")
def moe_permute_quant_int8(x, order):
    if _lib.native_path():
        done = _lib.native.int8_quant(x, order.rows, False)
        if done is not None:
            return done
    _one_device("moe_permute_quant_int8", x, order.rows)
    tokens, k = _pairs("moe_permute_quant_int8", order)
    if x.dim() != 2 or x.shape[0] != tokens:
        raise ValueError(f"moe_permute_quant_int8: x must have a row for each of {tokens} tokens, got {tuple(x.shape)}")
    q = torch.empty((tokens * k, x.shape[1]), dtype=torch.int8, device=x.device)
    scales = torch.empty(tokens * k, dtype=torch.float32, device=x.device)
    _lib.int8_quant(q, scales, x, order.rows)
    return q, scales


@register_impl("moe_unpermute", backend="hip")
def moe_unpermute(x, order, weights=None):
    if torch.is_grad_enabled() and (x.requires_grad or (weights is not None and weights.requires_grad)):
        _without_tangents("moe_unpermute", x, weights)
        _recordable("moe_unpermute", x, weights)
        if _lib.native_path():
            done = _lib.native.moe_unpermute_grad(x, order.rows, weights)
            if done is not None:
                return done
        return _Unpermute.apply(x, weights, *order)
    return _unpermute(x, order, weights)


@register_impl("moe_permute_backward", backend="hip")
def moe_permute_backward(grad_rows, order):
    return _unpermute(grad_rows.contiguous(), order, None, "moe_permute_backward")


@register_impl("moe_unpermute_backward", backend="hip")
def moe_unpermute_backward(grad_out, x, order, weights):
    grad_out = grad_out.contiguous()
    if _lib.native_path():
        done = _lib.native.moe_unpermute_backward(grad_out, x, order.rows, weights)
        if done is not None:
            return done
    _without_tangents("moe_unpermute_backward", grad_out, x, weights)
    _one_device("moe_unpermute_backward", grad_out, x, order.rows, weights)
    grad_x, grad_weights = torch.empty(x.shape, dtype=x.dtype, device=x.device), torch.empty(weights.shape, dtype=weights.dtype, device=x.device)
    _lib.moe_unpermute_backward(grad_x, grad_weights, grad_out, x, order.rows, weights)
    return grad_x, grad_weights
