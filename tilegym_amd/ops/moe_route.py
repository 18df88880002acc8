"""Tokens sorted by expert, carried to the experts' rows and back with the router's weights, and the gradients of both ways: what makes the
segments that ``ragged_block_scaled_bmm`` and ``ragged_int8_matmul`` multiply.

Gradients are those of reverse mode, and once: dual tensors are refused here and in the backward operators, and so are second derivatives.

Forward and backward passes can be captured into a graph.  What is refused while capturing is a leaf that an eager graph on another stream still holds: its gradient would be
added there (``moe_permute_backward`` and ``moe_unpermute_backward`` take no part in autograd and can always be captured).

The reference sorts inside ``moe_align_block_size`` (src/tilegym/ops/moe_interface.py:21-79), into blocks that its gather GEMM pads."""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from ..backend import dispatch, get_current_backend


class MoeOrder(NamedTuple):
    """The order of a routing's (token, slot) pairs by expert, all int32 on the device; every pair has a row and every row a pair.

    indptr (E + 1): rows indptr[e] : indptr[e + 1] belong to expert e.  rows (T, k): the row of each pair; where the pair's expert is not here (its id is
    outside [0, E)), -1 - row, and that row lies behind indptr[E].  slots (T * k): the pair of each row (token slots // k)."""

    indptr: torch.Tensor
    rows: torch.Tensor
    slots: torch.Tensor


@dispatch("moe_sort")
def moe_sort(topk_ids: torch.Tensor, num_experts: int) -> MoeOrder:
    """The order of topk_ids (T, k), int32 or int64, by expert; pairs of one expert keep their order.  One launch, or two for many pairs; nothing is
    read by the host.
    At most 512 experts."""
    raise NotImplementedError(f"moe_sort is not implemented for this backend: {get_current_backend()}")


@dispatch("moe_permute_backward")
def moe_permute_backward(grad_rows: torch.Tensor, order: MoeOrder) -> torch.Tensor:
    """The gradient of ``moe_permute``: (T, H) from grad_rows (T * k, H); a token's rows are summed in fp32, in the order of its slots, and rounded once.
    Rows of pairs without an expert add nothing."""
    raise NotImplementedError(f"moe_permute_backward is not implemented for this backend: {get_current_backend()}")


@dispatch("moe_unpermute_backward")
def moe_unpermute_backward(grad_out: torch.Tensor, x: torch.Tensor, order: MoeOrder, weights: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """The gradients of ``moe_unpermute`` with weights: (grad_x, grad_weights) from grad_out (T, H).  grad_x is weight * grad_out in the pair's row, and
    zero in the rows of pairs without an expert; grad_weights[t, j] is <grad_out[t], x[row]> summed in fp32, zero for those pairs."""
    raise NotImplementedError(f"moe_unpermute_backward is not implemented for this backend: {get_current_backend()}")


@dispatch("moe_permute")
def moe_permute(x: torch.Tensor, order: MoeOrder) -> torch.Tensor:
    """Each token's row of x (T, H), bf16 / f16 / fp32, contiguous, in the rows of its pairs: (T * k, H), sorted by expert.  The rows of pairs without an expert,
    behind indptr[E], are zeros.  Differentiable in x (by ``moe_permute_backward``)."""
    raise NotImplementedError(f"moe_permute is not implemented for this backend: {get_current_backend()}")


@dispatch("moe_permute_quant_int8")
def moe_permute_quant_int8(x: torch.Tensor, order: MoeOrder) -> Tuple[torch.Tensor, torch.Tensor]:
    """``quant_int8`` of x (T, H), contiguous, carried to the rows of each token's pairs: (q (T * k, H) int8, scales (T * k) fp32), in one launch.  The rows of pairs
    without an expert have codes of zero and a scale of 1."""
    raise NotImplementedError(f"moe_permute_quant_int8 is not implemented for this backend: {get_current_backend()}")


@dispatch("moe_unpermute")
def moe_unpermute(x: torch.Tensor, order: MoeOrder, weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Back to the tokens: out[t] = sum_j weights[t, j] * x[row of (t, j)], x (T * k, H) bf16 / f16 / fp32, weights (T, k) fp32 / bf16 / f16, or ones; all contiguous.
    Summed in fp32, in the order of the slots, rounded once.  Pairs without an expert add nothing, whatever their rows and weights hold.
    Differentiable in x and weights (by ``moe_unpermute_backward``, which makes both gradients whichever is asked for)."""
    raise NotImplementedError(f"moe_unpermute is not implemented for this backend: {get_current_backend()}")
