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
};
__device__ __forceinline__ SeqItem find_sequence(const int* __restrict__ indptr, int batch, int rows, int item, int num, int den, int more) {
    const int lane = (int)threadIdx.x & 63;
    int seq = -1;
    for (int base = 0; base < batch; base += 64) {
        const int b = base + lane;
        bool begun = false;
        if (b < batch) begun = (int)((int64_t)clamp_row(indptr[b], rows) * num / den) + more * b <= item;
        const int count = __popcll(__ballot(begun));
        seq += count;
        if (count < 64) break;
    }
    SeqItem f;
    f.seq = seq;
    f.first = f.n = f.item = 0;
    if (seq < 0) return f;
    f.first = clamp_row(indptr[seq], rows);
    f.n = clamp_row(indptr[seq + 1], rows) - f.first;
    f.item = item - ((int)((int64_t)f.first * num / den) + more * seq);
    if (f.n <= 0 || f.item < 0) f.seq = -1;
    return f;
}

}  // namespace tg
