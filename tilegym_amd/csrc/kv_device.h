// The paged e4m3 cache of keys and values, as its kernels see it.
//
//   k (pages, heads, P, D)   a token's D elements together: the rows of a matrix product over D
//   v (pages, heads, D, P)   transposed, an element's P tokens together: the rows of a matrix product over tokens.  16 tokens of an
//                            element are one 16-byte load, the operand of two matrix instructions without a shuffle
//   one fp32 scale per page and head for each half; element = code * scale
// Position p of sequence b lies in slot p % P of page table[b][p / P].  The new tokens of sequence b are rows
// indptr[b] .. indptr[b + 1] of the packed inputs and the last positions below lens[b].
// Every index that comes from device memory is checked before it is used as one: rows against the packed inputs, positions
// against the table's width, pages against the pool.  What lies outside is left out, whatever the tensors hold.
#pragma once
#include "tg_host.h"

namespace tg {

__device__ __forceinline__ int clamp_row(int x, int rows) { return min(max(x, 0), rows); }

// Which sequence work item `item` belongs to.  Sequence b's items begin at floor(indptr[b] * num / den) + more * b; the caller
// chooses num, den and more so that a sequence has at most as many items as lie between that and the next one's beginning, so no
// prefix sum over the sequences is needed: the last beginning that is not above `item`, by a ballot over 64 sequences at a
// time.  All lanes of a wave return the same.
struct SeqItem {
    int seq;        // -1: none
    int first, n;   // rows of the packed inputs
    int item;       // item of the sequence
    int len;        // its length, not below zero (0 without lens)
};
// All that is asked for comes in one round of loads: the neighbouring entry and the length by the lane that then turns out to have them.
__device__ __forceinline__ SeqItem find_sequence(const KvCache& c, int item, int num, int den, int more) {
    const int lane = (int)threadIdx.x & 63;
    SeqItem f;
    f.seq = -1, f.first = f.n = f.item = f.len = 0;
    for (int base = 0; base < c.batch; base += 64) {
        const int b = base + lane, at = min(b, c.batch - 1);
        const int first = clamp_row(c.indptr[at], c.rows), end = clamp_row(c.indptr[at + 1], c.rows), len = c.lens ? c.lens[at] : 0;
        const int begin = (int)((int64_t)first * num / den) + more * b;
        const int count = __popcll(__ballot(b < c.batch && begin <= item));
        if (count > 0) {
            f.seq = base + count - 1;
            f.first = __builtin_amdgcn_readlane(first, count - 1);
            f.n = __builtin_amdgcn_readlane(end, count - 1) - f.first;
            f.item = item - __builtin_amdgcn_readlane(begin, count - 1);
            f.len = max(__builtin_amdgcn_readlane(len, count - 1), 0);
        }
        if (count < 64) break;
    }
    if (f.n <= 0 || f.item < 0) f.seq = -1;
    return f;
}

// find_sequence for at most 64 sequences of at most one item each, the longest sequence first (of equal ones the first): item -1 where
// some sequence has more than one.  A lane's sequence is ranked by comparison with all others, a share of them in each of the
// workgroup's waves (WAVES; all of them call this).  part: LDS.
template <int WAVES>
__device__ __forceinline__ SeqItem find_longest(const KvCache& c, int item, int num, int den, int (*part)[64]) {
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), at = min(lane, c.batch - 1);
    const int first = clamp_row(c.indptr[at], c.rows), n = clamp_row(c.indptr[at + 1], c.rows) - first, len = max(c.lens[at], 0);
    int rank = 0;
#pragma unroll
    for (int i = 0; i < 64 / WAVES; ++i) {
        const int b = wave * (64 / WAVES) + i, other = __builtin_amdgcn_readlane(len, b);
        rank += b < c.batch && (other > len || (other == len && b < lane)) ? 1 : 0;
    }
    part[wave][lane] = rank;
    __syncthreads();
    rank = 0;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) rank += part[i][lane];
    SeqItem f;
    f.seq = -1, f.first = f.n = f.item = f.len = 0;
    if (__ballot((int64_t)n * num > den)) {
        f.item = -1;
        return f;
    }
    const uint64_t found = __ballot(lane < c.batch && rank == item);
    if (!found) return f;
    f.seq = __ffsll((unsigned long long)found) - 1;
    f.first = __builtin_amdgcn_readlane(first, f.seq), f.n = __builtin_amdgcn_readlane(n, f.seq), f.len = __builtin_amdgcn_readlane(len, f.seq);
    if (f.n <= 0) f.seq = -1;
    return f;
}

// A value that all lanes have alike, through the scalar cache: it is then not counted among the vector loads in flight
__device__ __forceinline__ int uniform_load(const int* at) { return *(const __attribute__((address_space(4))) int*)(uintptr_t)at; }
__device__ __forceinline__ float uniform_load(const float* at) { return *(const __attribute__((address_space(4))) float*)(uintptr_t)at; }

}  // namespace tg
