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

struct SeqItem {
    int seq;        // -1: none
    int first, n;   // rows of the packed inputs
    int item;       // item of the sequence
    int len;        // its length, not below zero (0 without lens)
};

// Inclusive prefix sum over the lanes of a wave, by lane permutations inside the vector instructions.
__device__ __forceinline__ int wave_prefix(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);  // row_shr 1, 2, 4, 8: inside rows of 16
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // row_bcast 15: a row's sum to the next, in rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // row_bcast 31: the lower half's to the upper
    return x;
}

// Which sequence work item `item` belongs to, where sequence b has count(n, len) items (n new rows of it, length len): 64 sequences at a time by a
// prefix sum over the lanes.  Items are numbered without gaps: workgroups without work in between would keep later ones waiting for
// the compute unit that they were dealt (256 workgroups of a compute unit each among 416: 29 us, without gaps 18).  from_end: item 0 is
// the last.  All that is asked for comes in one round of loads.  All lanes of a wave return the same.
template <typename Count>
__device__ __forceinline__ SeqItem find_sequence(const KvCache& c, int item, Count count, bool from_end = false) {
    const int lane = (int)threadIdx.x & 63;
    SeqItem f;
    f.seq = -1, f.first = f.n = f.item = f.len = 0;
    int first, n, len, items, prefix;
    auto load = [&](int base, int before) {
        const int b = base + lane, at = min(b, c.batch - 1);
        first = clamp_row(c.indptr[at], c.rows), n = clamp_row(c.indptr[at + 1], c.rows) - first, len = c.lens ? max(c.lens[at], 0) : 0;
        items = b < c.batch && n > 0 ? count(n, len) : 0;
        prefix = wave_prefix(items) + before;
        return __builtin_amdgcn_readlane(prefix, 63);
    };
    int total = load(0, 0);
    if (from_end) {
        for (int base = 64; base < c.batch; base += 64) total = load(base, total);
        item = total - 1 - item;
        if (item < 0) return f;
        if (c.batch > 64) total = load(0, 0);
    }
    for (int base = 0;;) {
        if (item < total) {
            const int found = __popcll(__ballot(prefix <= item));
            f.item = item - (__builtin_amdgcn_readlane(prefix, found & 63) - __builtin_amdgcn_readlane(items, found & 63));
            f.first = __builtin_amdgcn_readlane(first, found & 63), f.n = __builtin_amdgcn_readlane(n, found & 63);
            f.len = __builtin_amdgcn_readlane(len, found & 63);
            // (where indptr is no prefix sum, found may be anything: what it names is then checked against the tensors like the rest)
            if (found < 64 && base + found < c.batch && f.item >= 0 && f.n > 0) f.seq = base + found;
            return f;
        }
        base += 64;
        if (base >= c.batch) return f;
        total = load(base, total);
    }
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
