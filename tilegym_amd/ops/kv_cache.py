"""A paged cache of keys and values in e4m3 with one scale per page and head: writing it (with rotary positions), reading it back,
and attention over it: what lies between a layer's FP8 QKV projection and its output projection.

The reference's counterparts work on other caches: ``rope_quantize_fp8`` and the paged attention of its flashinfer suite
(src/tilegym/suites/flashinfer/), ``rope`` and flash decoding of ``tilegym.ops`` (src/tilegym/ops/ops.py:27-1040)."""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from ..backend import dispatch, get_current_backend

PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128, 256)


class KVCache(NamedTuple):
    """Tensors of a paged cache; an element is its code times its page's scale for that head.

    k (pages, heads, P, D) and v (pages, heads, D, P) float8_e4m3fn; k_scale and v_scale (pages, heads) fp32; all contiguous.
    v is transposed inside a page: 16 tokens of an element lie in 16 consecutive bytes, the operand of the matrix instructions that
    multiply by it.  Position p of sequence b is slot p % P of page ``block_table[b, p // P]``."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


def alloc_kv_cache(num_pages: int, num_kv_heads: int, head_dim: int, page_size: int = 64, device="cuda") -> KVCache:
    """An empty cache: page_size 16, 32, 64 or 128 tokens (a scale's block), head_dim 64, 128 or 256."""
    if page_size not in PAGE_SIZES or head_dim not in HEAD_DIMS:
        raise NotImplementedError(f"pages of {page_size} tokens, heads of {head_dim} elements are not implemented (pages of {PAGE_SIZES}, heads of {HEAD_DIMS})")
    fp8 = torch.float8_e4m3fn
    return KVCache(torch.zeros((num_pages, num_kv_heads, page_size, head_dim), dtype=torch.uint8, device=device).view(fp8),
                   torch.zeros((num_pages, num_kv_heads, head_dim, page_size), dtype=torch.uint8, device=device).view(fp8),
                   torch.ones((num_pages, num_kv_heads), dtype=torch.float32, device=device),
                   torch.ones((num_pages, num_kv_heads), dtype=torch.float32, device=device))


def rope_table(max_positions: int, rotary_dim: int, base: float = 10000.0, inv_freq: Optional[torch.Tensor] = None, position_scale: float = 1.0,
               magnitude: float = 1.0, device="cuda") -> torch.Tensor:
    """(max_positions, rotary_dim) fp32: a row holds the cosines of its position's rotary_dim / 2 angles, then the sines.

    The angle of pair i at position p is p * position_scale * inv_freq[i]; inv_freq is base^(-2 i / rotary_dim) unless given.  Angles
    are computed in float64: at position 10^6 a float32 angle is off by hundredths.  Scalings for long contexts are a
    ``position_scale`` below 1 (interpolation), another ``base``, or frequencies of one's own, with cosines and sines times
    ``magnitude`` where the rule asks for it."""
    if rotary_dim % 2 != 0:
        raise ValueError(f"rotary_dim must be even, got {rotary_dim}")
    if inv_freq is None:
        inv_freq = float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    elif inv_freq.numel() != rotary_dim // 2:
        raise ValueError(f"inv_freq must have {rotary_dim // 2} elements, got {inv_freq.numel()}")
    position = torch.arange(max_positions, dtype=torch.float64, device=device) * float(position_scale)
    angle = position[:, None] * inv_freq.reshape(1, -1).to(device=device, dtype=torch.float64)
    return (torch.cat([angle.cos(), angle.sin()], 1) * float(magnitude)).float()


@dispatch("kv_cache_append")
def kv_cache_append(
    cache: KVCache,
    k: torch.Tensor,
    v: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    indptr: torch.Tensor,
    q: Optional[torch.Tensor] = None,
    rope: Optional[torch.Tensor] = None,
    interleaved: bool = False,
) -> Optional[torch.Tensor]:
    """Write the new tokens' k and v (tokens, kv heads, D), bf16 or f16, into the cache, in place, in one launch.

    Rows indptr[b] : indptr[b + 1] are the last positions of sequence b, which has seq_lens[b] tokens with them; ``block_table``
    (B, width), ``seq_lens`` (B) and ``indptr`` (B + 1) are int32 on the device and are not read by the host.  Row and head
    strides are free (multiples of 8 elements): slices of a QKV projection's output need no copy.

    ``rope`` (a ``rope_table`` of at least width * page size positions): k's first rotary_dim elements are turned by the angles of the
    token's position, in pairs (i, i + rotary_dim / 2), or (2 i, 2 i + 1) if ``interleaved``; rotary_dim a multiple of 16.  ``q``
    (tokens, any number of heads, D) is then turned too, and returned as a new tensor.

    A page's scale for a head is a power of two, 2^e with the smallest e in [-40, 40] that brings the page's largest magnitude
    within 448; beyond 448 * 2^40 and at infinities codes saturate; NaN becomes -448, as in ``act_quant``.  Writing a page from its first slot on
    sets its scale anew.  Writing behind earlier tokens keeps the larger of the page's scale and the new tokens' and moves the
    earlier codes to it, which is exact except where they become subnormal.

    Pages are written by one sequence at a time: no page twice in what a call writes.  Positions beyond the table's width and pages outside
    the pool (such as -1) are not written; q of positions below zero or beyond ``rope`` is turned by its first or last row.  Rows of no sequence:
    their q is left unwritten."""
    raise NotImplementedError(f"kv_cache_append is not implemented for this backend: {get_current_backend()}")


@dispatch("kv_cache_read")
def kv_cache_read(
    cache: KVCache,
    block_table: torch.Tensor,
    indptr: torch.Tensor,
    total_tokens: int,
    out_dtype: torch.dtype = torch.bfloat16,
    k_out: Optional[torch.Tensor] = None,
    v_out: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """The first indptr[b + 1] - indptr[b] tokens of every sequence b as rows: (k, v), each (total_tokens, kv heads, D) of ``out_dtype``
    (bf16 / f16 / fp32), code times scale rounded once.  ``total_tokens`` is the host's number of rows, at least indptr[-1]; rows of no
    sequence, and of tokens whose page is not in the pool, are left as they were in ``k_out`` / ``v_out``, and unset without them."""
    raise NotImplementedError(f"kv_cache_read is not implemented for this backend: {get_current_backend()}")


@dispatch("kv_cache_attention")
def kv_cache_attention(
    q: torch.Tensor,
    cache: KVCache,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    indptr: torch.Tensor,
    sm_scale: Optional[float] = None,
    window: int = 0,
    sink_tokens: int = 0,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Causal attention of the new tokens' q (tokens, heads, D), bf16 or f16, over the cache that already holds them.

    ``block_table``, ``seq_lens`` and ``indptr`` as in ``kv_cache_append``: one new token per sequence is decoding, a few are the check of
    drafted ones, many are a prompt or a chunk of one; they may be mixed.  heads is a multiple of the cache's: query head h reads
    cache head h // (heads // kv heads).  ``sm_scale`` defaults to D^-1/2.  Row and head strides of q are free (multiples of 8 elements).

    A token sees the positions up to its own; with ``window`` > 0 only the last ``window`` of them (its own included) and the
    first ``sink_tokens`` of the sequence.  Pages that no token sees need not exist (their table entries may be -1).  A
    token that sees nothing gets zeros; one whose scores are no numbers (NaN or infinities in q) gets no numbers; one behind the table's
    end sees the positions that the table has.  Scores, the softmax's maximum and sum and the results are held in fp32; the softmax's weights times
    their values' page scales are rounded to q's 16-bit type in front of the product with v's codes, by up to 2^-8 of their own size in bf16, 2^-11 in f16
    (there by up to 2^-32 of the row's largest where that is more), and the result once more.  Results do not depend on what unwritten slots hold, and a call gives the same bits every time.

    Returns (tokens, heads, D) of q's type; ``out`` (contiguous, not q) is written if given.  Rows of no sequence are left as they were
    in ``out``, and unset without it."""
    raise NotImplementedError(f"kv_cache_attention is not implemented for this backend: {get_current_backend()}")
