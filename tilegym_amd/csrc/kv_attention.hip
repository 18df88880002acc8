// Causal attention of new tokens over the paged e4m3 cache (kv_device.h), whole or in a window with a few first tokens visible:
//   O_i = sum_j softmax_j(c q_i . k_j) v_j  over j <= p_i with p_i - j < window or j < sinks,  k = code * k_scale, v = code * v_scale
// The query heads of one key/value head share its keys: row r of a sequence is token r / group, head r % group of the group, and a tile of
// rows runs over the keys together, whatever the tokens and the group are.
//
// One pass over the keys in steps of 64, with the running maximum m and sum l of the softmax (fp32, in powers of two).  Both products run on 16x16x32 matrix
// instructions with the tile's rows as columns:
//   S^T (keys x rows) = K Q^T;   O^T (elements x rows) += V^T P^T
// so a lane's scores all belong to one row (column lane % 16): no shuffle for P, m's reduction goes over 4 lanes only, and O is
// rescaled lane by lane.  The key that a row of the first product stands for is free to choose: row 4 g + i of step t takes key 16 g + 4 t + i, so
// that lane group g ends up with the 16 consecutive keys 16 g ... of its row.  Those are, in order, the second product's operand, and
// the cache's transposed v has them in 16 consecutive bytes.  They lie in one page (P is a multiple of 16), so scales are
// one value per lane.
// Codes become the 16-bit type of q exactly (e4m3 has 4 significant bits).  k's scale joins the softmax's factor.  v's scale joins the softmax's
// exponent: m is the maximum of a row's c q.k + log2 v_scale, and P, rounded to 16 bits, is exp2 of that less m (off by 2^-8 relative in bf16, 2^-11 in f16, of its own value,
// in f16 by no more than 2^-32 of the row's largest where that is more).  S, m, l and O are fp32.
//
// What is not seen is taken out by selection, never by arithmetic: scores before the maximum, and v's codes, since 0 x NaN is NaN
// and a page's unwritten slots may hold anything.
#include "kv_device.h"

#include <algorithm>
#include <type_traits>

namespace tg {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

typedef float v16f __attribute__((ext_vector_type(16)));

template <typename T> struct Types;
template <> struct Types<__bf16> { typedef bf16x8 v8; typedef bf16x2 v2; };
template <> struct Types<_Float16> { typedef f16x8 v8; typedef f16x2 v2; };

__device__ __forceinline__ v4f mfma16(bf16x8 a, bf16x8 b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ v4f mfma16(f16x8 a, f16x8 b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

__device__ __forceinline__ v16f mfma32(bf16x8 a, bf16x8 b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ v16f mfma32(f16x8 a, f16x8 b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// eight e4m3 codes -> T, exact
template <typename T>
__device__ __forceinline__ typename Types<T>::v8 widen(int lo, int hi) {
    typename Types<T>::v2 a, b, c, d;
    if constexpr (std::is_same_v<T, __bf16>) {
        a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
        c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
    } else {
        a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
        c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
    }
    return __builtin_shufflevector(__builtin_shufflevector(a, b, 0, 1, 2, 3), __builtin_shufflevector(c, d, 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
}

constexpr int kComputeUnits = 256;
constexpr int kMostSplits = 64;
constexpr int kLeastSteps = 8;  // of a split

// A load through the vector path whatever the address is
template <typename X>
__device__ __forceinline__ X vector_load(const X* at) {
    int zero = 0;
    asm("" : "+v"(zero));
    return at[zero];
}

constexpr float kMinusInf = -__builtin_inff();
// The maximum that a row's scores are taken against is looked for only when 16 weights against the old one add up to more than this: floating
// point loses no precision in weights above 1 (f16 holds 16 times as much, and sums and O are fp32; a maximum's 16 weights are 2048 at most).  A row's first keys find a maximum of
// -inf and so a sum that is not a number, and take the same path.  In the other steps there is no search, no exchange between lanes
// and no rescaling of O.
constexpr float kLargeSum = 4096.f;

// 16 bytes per lane from memory to LDS without a register between: lane i's go to lds_addr + 16 i.  Inline assembly, as the compiler would have every
// later LDS read wait for a direct load in flight; the kernel waits itself, in front of the barrier after which they are read.  The
// write of M0 and the s_nop are the five wait states that a scalar operand written by a vector instruction needs.
__device__ __forceinline__ void load_to_lds(uint32_t lds_addr, const uint8_t* base, uint32_t offset) {  // base: a scalar
    lds_addr = __builtin_amdgcn_readfirstlane(lds_addr);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(lds_addr), "v"(offset), "s"(base) : "memory");
}
__device__ __forceinline__ void load_to_lds(uint32_t lds_addr, const uint8_t* at) {
    lds_addr = __builtin_amdgcn_readfirstlane(lds_addr);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(lds_addr), "v"(at) : "memory");
}
__device__ __forceinline__ uint32_t lds_address(const void* p) { return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p; }

// The rows of one workgroup and the steps of 64 keys that any of them sees.  Positions and keys are below 2^30 (the table's capacity)
// or a sequence's length.
struct RowTile {
    int seq, head;          // sequence, key/value head
    int first, r0, rows;    // sequence's first packed row; the tile's first row of the sequence, and how many it has
    int start;              // position of the sequence's first new token
    int low, high;          // positions of the tile's first and last row
    int key0, key1;         // keys [key0, key1) and, below key0, [0, sinks)
    int steps, sink_steps;  // steps of 64 keys: sink_steps from 0 on, then from key0 / 64 on
    __device__ __forceinline__ int key_of(int step) const { return (step < sink_steps ? step : (key0 >> 6) + step - sink_steps) * 64; }
};

// Tiles of ROWS rows of a sequence with n new tokens.
template <int ROWS>
__device__ __forceinline__ auto tiles_of(int group) {
    return [group](int n, int) { return (int)(((int64_t)n * group + ROWS - 1) / ROWS); };
}

__device__ __forceinline__ bool set_tile(const KvAttentionParams& p, const SeqItem& f, int tile_rows, int head, RowTile& t) {
    const KvCache& c = p.c;
    if (f.seq < 0) return false;
    const int64_t r0 = (int64_t)f.item * tile_rows, total = (int64_t)f.n * p.group;
    if (r0 >= total) return false;
    t.seq = f.seq, t.head = head, t.first = f.first;
    t.r0 = (int)r0, t.rows = (int)min((int64_t)tile_rows, total - r0);
    t.start = f.len - f.n;
    t.low = t.start + t.r0 / p.group, t.high = t.start + (t.r0 + t.rows - 1) / p.group;
    const int capacity = c.width << c.page_log2;
    t.key1 = t.high < 0 ? 0 : t.high < capacity ? t.high + 1 : capacity;
    t.key0 = p.window ? (int)min(max((int64_t)t.low - (p.window - 1), (int64_t)0), (int64_t)t.key1) : 0;  // (positions may lie below zero)
    const int sinks = min(p.sinks, t.key0);
    t.sink_steps = min((sinks + 63) >> 6, t.key0 >> 6);
    t.steps = t.key1 > 0 ? t.sink_steps + (((t.key1 + 63) >> 6) - (t.key0 >> 6)) : 0;
    return true;
}

// The table's entry for the page of 16 keys, as it is: looked at a step later (page_of), so that the load is not waited for.
__device__ __forceinline__ int table_entry(const KvCache& c, const int* row, int key) { return vector_load(row + min(key >> c.page_log2, c.width - 1)); }
// A page, or one that may be read in its place (its keys are then not seen).
struct Granule {
    int page;
    bool there;
};
__device__ __forceinline__ Granule page_of(const KvCache& c, int entry) {
    Granule g;
    g.there = entry >= 0 && entry < c.pages;
    g.page = g.there ? entry : 0;
    return g;
}
// The same for 16 keys from `key` on, which may lie behind the table's end: a table of pages of 16 or 32 can end inside a step of 64 keys, and
// table_entry then gives its last page.  (Positions behind the end are possible too: they see what the table has.)
__device__ __forceinline__ Granule page_of(const KvCache& c, int entry, int key) {
    Granule g = page_of(c, entry);
    g.there = g.there && (key >> c.page_log2) < c.width;
    return g;
}

// Bytes of 16 codes of v that some row sees: those of keys first .. first + 15 that lie in [key0, key1) or among the sinks, all or none
// towards the lower end (earlier keys of the same page are numbers), and exactly towards the upper (later slots may hold anything).
__device__ __forceinline__ v4i seen_codes(v4i codes, const RowTile& t, int sinks, int first, bool there) {
    const bool any = there && first < t.key1 && (first + 16 > t.key0 || first < sinks);
    const int live = any ? t.key1 - first : 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const int bytes = min(max(live - 4 * w, 0), 4);
        codes[w] &= bytes == 4 ? -1 : (1 << (8 * bytes)) - 1;
    }
    return codes;
}

// A lane's 16 scores: four results of a 16 x 16 product, or one of a 32 x 32
struct Scores16 {
    v4f x[4];
    __device__ __forceinline__ float operator[](int i) const { return x[i / 4][i % 4]; }
    __device__ __forceinline__ void set(int i, float f) { x[i / 4][i % 4] = f; }
    static constexpr int kFirstLane = 16;  // lanes this far apart, and the further powers of two, share a row
};
struct Scores32 {
    v16f x;
    __device__ __forceinline__ float operator[](int i) const { return x[i]; }
    __device__ __forceinline__ void set(int i, float f) { x[i] = f; }
    static constexpr int kFirstLane = 32;
};

template <typename S>
__device__ __forceinline__ void select_seen(S& s, int key, int position, int window, int sinks, bool there) {
    const int first_seen = window ? position - (window - 1) : 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int j = key + i;
        const bool seen = there && j <= position && (j >= first_seen || j < sinks);
        s.set(i, seen ? s[i] : kMinusInf);
    }
}

// v's scale in a lane's 16 keys of a step: it joins the weight's exponent, so that P is p v_scale against the row's largest such product so far (2^m), and
// is taken out of the sum again.  What 16 bits lose of a weight is then measured by what the row itself adds up, whatever scales other rows and
// pages without weight have.  In f16 weights stand 128 times as high: one that f16's smallest step swallows is below 2^-32 of the row's largest
// product and not 2^-25, which tens of thousands of faint keys beside one strong one would add up to more than a rounding of the result.  Times a
// code it is at most 2^-23 of the largest product; e4m3 itself rounds that key's value by up to 2^-10 of it, or more.
// With q in bf16 P is bf16, which has no such end: where the heaviest keys' values are zero in an element, the faint keys' are still held to 2^-8.  f16 weights there
// lose those, though they are nearer to 64 bits elsewhere (4096 tokens over 1500 to 4500 keys: relative error 0.0016 and 0.0022; 182 and 174 us).
template <typename T>
struct ValueScale {
    static constexpr int kUp = std::is_same_v<T, __bf16> ? 0 : 7;
    static constexpr float kDown = 1.f / (1 << kUp);  // O is held in units of 2^m kDown
    float log, back;
    // seen: whether any key of the lane's 16 is seen (the scale of the others may be anything).  Scales are 2^-40 to 2^40 as written; others are held
    // within what fp32 sums of 1 / scale can take
    __device__ __forceinline__ void set(float v_scale, bool seen) {
        const float s = __builtin_amdgcn_fmed3f(seen ? v_scale : 1.f, 0x1p-64f, 0x1p100f);
        log = __builtin_amdgcn_logf(s), back = __builtin_amdgcn_rcpf(s) * kDown;
    }
};

// One row's 16 scores of a step -> its weights against the running maximum m, and its sum l of exp2(score - m).  Returns what O has to
// be multiplied by on m's account.  factor > 0.
template <typename T, typename S>
__device__ __forceinline__ float weigh(const S& s, float factor, const ValueScale<T>& v, float& m, float& l, typename Types<T>::v8 (&pt)[2]) {
    v16f w;
    const float lift = v.log + (float)ValueScale<T>::kUp;
    float shrink = 1.f, base = lift - m, sum = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], factor, base));
        sum = i == 0 ? w[i] : sum + w[i];
    }
    if (__ballot(!(sum <= kLargeSum))) {
        float top = kMinusInf;
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[i] * factor);
        top += v.log;
#pragma unroll
        for (int d = S::kFirstLane; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
        top = fmaxf(m, top);
        const float finite = top == kMinusInf ? 0.f : top;
        shrink = __builtin_amdgcn_exp2f(m - finite);
        l *= shrink;
        m = top;
        base = lift - finite;
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], factor, base));
            sum += w[i];
        }
    }
    l = __builtin_fmaf(sum, v.back, l);
    pt[0] = __builtin_convertvector(__builtin_shufflevector(w, w, 0, 1, 2, 3, 4, 5, 6, 7), typename Types<T>::v8);
    pt[1] = __builtin_convertvector(__builtin_shufflevector(w, w, 8, 9, 10, 11, 12, 13, 14, 15), typename Types<T>::v8);
    return shrink;
}

// q's eight elements with the softmax factor's sign, which the scores then need not have
template <typename T>
__device__ __forceinline__ typename Types<T>::v8 load_q(const T* at, bool negative) {
    v4i x = *reinterpret_cast<const v4i*>(at);
    if (negative) x ^= (int)0x80008000;
    return __builtin_bit_cast(typename Types<T>::v8, x);
}

// k's scale and the softmax factor; never zero, so that what is not seen stays at -inf
__device__ __forceinline__ float score_factor(float k_scale, float scale_log2) { return fmaxf(fabsf(k_scale * scale_log2), 0x1p-126f); }

// Few rows: eight waves (four with 256 elements, which take the registers of two), 16 NT rows; the waves take the steps of the workgroup's share in
// turn and join at the end.  Codes come straight from memory into registers, k's of the next step being asked for when this step's are used
// up, v's likewise.  Bound by HBM once some 150 compute units have work (64 sequences of 100 to 8000 keys x 8 heads: 5.5 TB/s), by latency below
// that.  Eight waves and one workgroup to a compute unit against four and two: those 64 sequences, long ones first, 98 and 110 us; 64 of 4000 keys each
// 101 and 98, 8 of them 19.5 and 19.2, one of 777 11.4 and 10.3.  The forms of 16 rows keep 43 to 77 of their scalars in lanes of vector registers (the compiler's
// scalar spills); no vector register spills.
template <int D>
constexpr int kFewWaves = D == 256 ? 4 : 8;
// ONE: pages hold whole steps (64 or 128 tokens), so a step's page, its scales and its address are scalars.
template <typename T, int D, int NT, bool ONE>
__global__ void __launch_bounds__(64 * kFewWaves<D>, D == 256 ? 1 : 2) kv_attention_kernel(const KvAttentionParams p) {
    typedef typename Types<T>::v8 v8;
    constexpr int WAVES = kFewWaves<D>, CH = D / 64, DT = D / 16, ROWS = 16 * NT;  // 64-element chunks of a key, 16-element tiles of a value
    const KvCache& c = p.c;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, g = lane >> 4;
    const int split = (int)blockIdx.x % p.splits, rest = (int)blockIdx.x / p.splits;
    RowTile t;
    {
        __shared__ int ranks[WAVES][64];
        SeqItem f;
        f.item = -1;
        if (p.longest_first) f = find_longest<WAVES>(c, rest / c.heads, p.group, ROWS, ranks);
        if (f.item < 0) f = find_sequence(c, rest / c.heads, tiles_of<ROWS>(p.group));
        if (!set_tile(p, f, ROWS, rest % c.heads, t)) return;
    }
    const int share = p.splits == 1 ? t.steps : max((t.steps + p.splits - 1) / p.splits, kLeastSteps);
    const int begin = min(split * share, t.steps), end = min(begin + share, t.steps);

    const int P = 1 << c.page_log2, in_page = P - 1, head_bytes = P * D;
    const int* table = c.table + (int64_t)t.seq * c.width;
    const int k_key = 16 * (col >> 2) + (col & 3);  // this lane's first key of a step as a row of K, and 16 g its first as a column of V^T

    v4i kc[4][CH], vc[DT];
    int k_entry = 0, v_entry = 0;
    Granule v_page{0, false}, there{0, false};
    float k_scale = 0.f, v_scale = 0.f;
    auto load_pages = [&](int step) {
        if (step >= end) return;
        const int key = t.key_of(step);
        if constexpr (ONE) {
            v_entry = uniform_load(table + min(key >> c.page_log2, c.width - 1));
        } else {
            k_entry = table_entry(c, table, key + 16 * (col >> 2)), v_entry = table_entry(c, table, key + 16 * g);
        }
    };
    const int k_lane = k_key * D + g * 16, v_lane = col * P + 16 * g;
    auto load_k = [&](int step) {
        const int key = t.key_of(step);
        v_page = ONE ? page_of(c, v_entry) : page_of(c, v_entry, key + 16 * g);
        const int64_t at = (int64_t)v_page.page * c.heads + t.head;
        if constexpr (ONE) {
            const uint8_t* base = c.k + at * head_bytes + (key & in_page) * D;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int ch = 0; ch < CH; ++ch) kc[i][ch] = *reinterpret_cast<const v4i*>(base + (uint32_t)k_lane + (i * 4 * D + ch * 64));
            k_scale = uniform_load(c.k_scale + at);
        } else {
            const uint8_t* base = c.k + ((int64_t)page_of(c, k_entry).page * c.heads + t.head) * head_bytes + ((key + k_key) & in_page) * D + g * 16;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int ch = 0; ch < CH; ++ch) kc[i][ch] = *reinterpret_cast<const v4i*>(base + i * 4 * D + ch * 64);
            k_scale = c.k_scale[at];
        }
    };
    auto load_v = [&](int step) {
        there = v_page;
        const int key = t.key_of(step);
        const int64_t at = (int64_t)v_page.page * c.heads + t.head;
        if constexpr (ONE) {
            // (one scalar base: eight would not fit the scalar registers)
            const uint8_t* base = c.v + at * head_bytes;
            const int offset = v_lane + (key & in_page);
#pragma unroll
            for (int d = 0; d < DT; ++d) vc[d] = *reinterpret_cast<const v4i*>(base + (uint32_t)(offset + d * 16 * P));
            v_scale = uniform_load(c.v_scale + at);
        } else {
            const uint8_t* base = c.v + at * head_bytes + col * P + ((key + 16 * g) & in_page);
#pragma unroll
            for (int d = 0; d < DT; ++d) vc[d] = *reinterpret_cast<const v4i*>(base + d * 16 * P);
            v_scale = c.v_scale[at];
        }
    };
    const int mine = begin + wave;
    load_pages(mine);

    // this lane's rows
    int position[NT];
    v8 q[NT][CH][2];
    float m[NT], l[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int row = n * 16 + col, r = t.r0 + row, token = r / p.group, q_head = t.head * p.group + r % p.group;
        position[n] = row < t.rows ? t.start + token : -1;
        m[n] = row < t.rows ? kMinusInf : 0.f, l[n] = 0.f;
#pragma unroll
        for (int ch = 0; ch < CH; ++ch)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                q[n][ch][h] = v8{};
                if (row < t.rows) q[n][ch][h] = load_q<T>((const T*)p.q + (int64_t)(t.first + token) * p.q_row + (int64_t)q_head * p.q_head + ch * 64 + g * 16 + h * 8, p.scale_log2 < 0.f);
            }
    }
    if (mine < end) {
        load_k(mine);
        load_v(mine);
        load_pages(mine + WAVES);
    }
    v4f o[NT][DT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int d = 0; d < DT; ++d) o[n][d] = v4f{0.f, 0.f, 0.f, 0.f};

    for (int step = mine; step < end; step += WAVES) {
        const int key = t.key_of(step), first = key + 16 * g;
        Scores16 s[NT];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int n = 0; n < NT; ++n) s[n].x[i] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ch = 0; ch < CH; ++ch) {
                const v8 a = widen<T>(kc[i][ch][0], kc[i][ch][1]), b = widen<T>(kc[i][ch][2], kc[i][ch][3]);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    s[n].x[i] = mfma16(a, q[n][ch][0], s[n].x[i]);
                    s[n].x[i] = mfma16(b, q[n][ch][1], s[n].x[i]);
                }
            }
        }
        const float factor = score_factor(k_scale, p.scale_log2);
        if (step + WAVES < end) load_k(step + WAVES);
        // every key of the step seen by every row: nothing to select
        const bool whole = key + 63 <= t.low && (!p.window || key > t.high - p.window) && __ballot(!there.there) == 0;
        ValueScale<T> value;
        value.set(v_scale, whole || (there.there && first < t.key1 && (first + 16 > t.key0 || first < p.sinks)));
        if (!whole) {
#pragma unroll
            for (int n = 0; n < NT; ++n) select_seen(s[n], first, position[n], p.window, p.sinks, there.there);
#pragma unroll
            for (int d = 0; d < DT; ++d) vc[d] = seen_codes(vc[d], t, p.sinks, first, there.there);
        }
        v8 pt[NT][2];
        float rescale[NT];
        bool any = false;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            rescale[n] = weigh<T>(s[n], factor, value, m[n], l[n], pt[n]);
            any = any || rescale[n] != 1.f;
        }
        if (__ballot(any)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int d = 0; d < DT; ++d) o[n][d] *= rescale[n];
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const v8 a = widen<T>(vc[d][0], vc[d][1]), b = widen<T>(vc[d][2], vc[d][3]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                o[n][d] = mfma16(a, pt[n][0], o[n][d]);
                o[n][d] = mfma16(b, pt[n][1], o[n][d]);
            }
        }
        if (step + WAVES < end) {
            load_v(step + WAVES);
            load_pages(step + 2 * WAVES);
        }
    }

    // the waves' results: m and l, then O, each in units of the largest
    __shared__ float part_m[WAVES][ROWS], part_l[WAVES][ROWS];
    __shared__ float part_o[WAVES][16][D + 4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        l[n] += __shfl_xor(l[n], 16);
        l[n] += __shfl_xor(l[n], 32);
        if (lane < 16) part_m[wave][n * 16 + col] = m[n], part_l[wave][n * 16 + col] = l[n];
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        __syncthreads();
        float top = part_m[0][n * 16 + col];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) top = fmaxf(top, part_m[w][n * 16 + col]);
        const float base = top == kMinusInf ? 0.f : top, f = __builtin_amdgcn_exp2f(m[n] - base) * ValueScale<T>::kDown;
#pragma unroll
        for (int d = 0; d < DT; ++d) *reinterpret_cast<v4f*>(&part_o[wave][col][d * 16 + 4 * g]) = o[n][d] * f;
        __syncthreads();
        constexpr int QUADS = D / 4;
        const int rows = min(t.rows - n * 16, 16);
        for (int i = tid; i < rows * QUADS; i += 64 * WAVES) {
            const int row = i / QUADS, e = 4 * (i % QUADS), rr = t.r0 + n * 16 + row;
            float row_top = part_m[0][n * 16 + row];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) row_top = fmaxf(row_top, part_m[w][n * 16 + row]);
            const float row_base = row_top == kMinusInf ? 0.f : row_top;
            float sum = 0.f;
            v4f x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                sum += part_l[w][n * 16 + row] * __builtin_amdgcn_exp2f(part_m[w][n * 16 + row] - row_base);
                x += *reinterpret_cast<const v4f*>(&part_o[w][row][e]);
            }
            const int64_t out_row = (int64_t)(t.first + rr / p.group) * p.q_heads + t.head * p.group + rr % p.group;
            if (p.splits > 1) {
                const int64_t at = (int64_t)split * c.rows * p.q_heads + out_row;
                if (e == 0) p.part_ml[2 * at] = row_top, p.part_ml[2 * at + 1] = sum;
                if (!(sum == 0.f)) *reinterpret_cast<v4f*>(p.part_o + at * D + e) = x;
            } else {
                typedef T v4t __attribute__((ext_vector_type(4)));
                x *= sum == 0.f ? 0.f : 1.0f / sum;  // a row that sees nothing is zero; a sum that is no number shows
                *reinterpret_cast<v4t*>((T*)p.out + out_row * D + e) = __builtin_convertvector(x, v4t);
            }
        }
    }
}

// Many rows: 128 of them per workgroup, 32 per wave, and every wave runs over the same keys, whose codes go to LDS for all four
// without a register between, the next step's while this one's products run, in two buffers with one barrier a step.  Codes stay
// e4m3 in LDS (half the reads that 16 bits would cost) and are widened behind each read, for 32 rows.  Bound by the SIMDs' issue, products and the
// softmax's and widening's vector instructions sharing them, two waves each: 4096 tokens of 3 sequences x 32 heads over 1500 to 4500 keys 176 us, 880
// TFLOP/s (a large 16-bit product: 1205); with 16 bits in LDS 4 % more, with three waves per SIMD spills.
// The products are 32x32x16 instructions on 32 keys at a time, the same way round: S^T row 8 a + 4 h + b stands for key 16 h + 4 a + b, so a
// lane (row lane % 32, h = lane / 32) has 16 consecutive keys of its one row.
// 16-byte chunks lie in LDS so that the 8, and the 16, neighbouring lanes that read together cover different banks: chunk ^ f,
// f of bits 0, 1, 2 and 4 of k's row (its key), and of bits 1, 2 and 3 of v's row (its element).
template <int D>
__device__ __forceinline__ int k_swizzle(int key) {
    const int b0 = key & 1, b1 = (key >> 1) & 1, b2 = (key >> 2) & 1, b4 = (key >> 4) & 1;
    return D == 64 ? (b1 ^ b2) + 2 * b4 : D == 128 ? b1 + 2 * b4 + 4 * (b0 ^ b2) : b0 + 2 * b1 + 4 * b4 + 8 * b2;
}
__device__ __forceinline__ int v_swizzle(int row) { return (((row >> 1) ^ (row >> 3)) & 1) + 2 * ((row >> 2) & 1); }

template <typename T, int D, bool ONE>
__global__ void __launch_bounds__(256, D == 256 ? 1 : 2) kv_attention_rows_kernel(const KvAttentionParams p) {
    typedef typename Types<T>::v8 v8;
    constexpr int CH = D / 32, DT = D / 32, LOADS = D / 64, KCH = D / 16;  // 32-element chunks of a key, 32-element tiles of a value
    __shared__ __align__(16) uint8_t lds_k[2][64 * D], lds_v[2][64 * D];
    const KvCache& c = p.c;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, h = lane >> 5;
    const int head = (int)blockIdx.x % c.heads, rest = (int)blockIdx.x / c.heads, split = rest % p.splits;
    RowTile t;
    if (!set_tile(p, find_sequence(c, rest / p.splits, tiles_of<128>(p.group), true), 128, head, t)) return;  // (the last rows of a sequence, which see most, first)
    const int share = max((t.steps + p.splits - 1) / p.splits, kLeastSteps);
    const int begin = min(split * share, t.steps), end = min(begin + share, t.steps);

    const int P = 1 << c.page_log2, in_page = P - 1, head_bytes = P * D;
    const int* table = c.table + (int64_t)t.seq * c.width;
    // a step's pages (one for each 16 of a lane's keys, in each half of the step; with ONE one scalar), then its codes and scales on
    // their way to LDS.  A thread's loads: rows and chunks of its own, the same in every step
    // (256 threads on, v's row is 64 further, k's 4096 / D: the swizzle is the same, for k if that is a multiple of 32)
    constexpr int K_ROWS = 4096 / D;
    const int k_row = tid / KCH, v_chunk = (tid & 3) ^ v_swizzle(tid / 4), v_at0 = (tid / 4) * P + v_chunk * 16;
    int k_at[K_ROWS % 32 == 0 ? 1 : LOADS];
#pragma unroll
    for (int j = 0; j < (K_ROWS % 32 == 0 ? 1 : LOADS); ++j) k_at[j] = (k_row + j * K_ROWS) * D + ((tid % KCH) ^ k_swizzle<D>(k_row + j * K_ROWS)) * 16;
    auto k_offset = [&](int j) { return K_ROWS % 32 == 0 ? k_at[0] + j * K_ROWS * D : k_at[j]; };
    constexpr int HALVES = ONE ? 1 : 2;
    float k_scale[HALVES], v_scale[HALVES];
    int entry[HALVES];
    Granule there[HALVES];
    // (entries are asked for past the last step too: the index is kept inside the table's row)
    auto load_page = [&](int key) {
        entry[0] = table_entry(c, table, key + (ONE ? 0 : 16 * h));
        if constexpr (!ONE) entry[HALVES - 1] = table_entry(c, table, key + 32 + 16 * h);
    };
    const int64_t page_bytes = (int64_t)c.heads * head_bytes;
    const uint8_t *k_head = c.k + (int64_t)head * head_bytes, *v_head = c.v + (int64_t)head * head_bytes;
    auto load_codes = [&](int key, int buffer) {
        const uint32_t k_to = lds_address(&lds_k[0][0]) + buffer * (64 * D) + wave * 1024, v_to = lds_address(&lds_v[0][0]) + buffer * (64 * D) + wave * 1024;
        if constexpr (ONE) {
            // (vector loads, made scalar where they are used: scalar ones would be waited for by every LDS read)
            there[0] = page_of(c, __builtin_amdgcn_readfirstlane(entry[0]));
            const int64_t at = (int64_t)there[0].page * c.heads + head, offset = there[0].page * page_bytes;
            k_scale[0] = vector_load(c.k_scale + at), v_scale[0] = vector_load(c.v_scale + at);
            const uint8_t *k_base = k_head + (offset + (key & in_page) * D), *v_base = v_head + (offset + (key & in_page));
#pragma unroll
            for (int j = 0; j < LOADS; ++j) {
                if constexpr (K_ROWS % 32 == 0) load_to_lds(k_to + 4096 * j, k_base + j * K_ROWS * D, (uint32_t)k_at[0]);
                else load_to_lds(k_to + 4096 * j, k_base, (uint32_t)k_at[j]);
                load_to_lds(v_to + 4096 * j, v_base + j * 64 * P, (uint32_t)v_at0);
            }
        } else {
#pragma unroll
            for (int i = 0; i < HALVES; ++i) {
                there[i] = page_of(c, entry[i], key + 32 * i + 16 * h);
                const int64_t at = (int64_t)there[i].page * c.heads + head;
                k_scale[i] = c.k_scale[at], v_scale[i] = c.v_scale[at];
            }
            auto block = [&](int sixteenth) {  // of 16 keys: held by the lanes of one h, as entry of one half
                const int lo = __shfl(there[0].page, (sixteenth & 1) * 32), hi = __shfl(there[HALVES - 1].page, (sixteenth & 1) * 32);
                return (sixteenth < 2 ? lo : hi) * page_bytes;
            };
#pragma unroll
            for (int j = 0; j < LOADS; ++j)
                load_to_lds(k_to + 4096 * j, k_head + block((k_row + j * K_ROWS) >> 4) + (((key + k_row + j * K_ROWS) & in_page) * D + (k_offset(j) & (D - 1))));
            const uint8_t* v_from = v_head + block(v_chunk) + ((tid / 4) * P + ((key + 16 * v_chunk) & in_page));
#pragma unroll
            for (int j = 0; j < LOADS; ++j) load_to_lds(v_to + 4096 * j, v_from + j * 64 * P);
        }
    };
    // the keys of this step, the next and the one after it
    auto key_behind = [&](int key, int step) { return step == t.sink_steps ? t.key0 & ~63 : key + 64; };  // step: the one behind
    int key = t.key_of(begin), key1 = key_behind(key, begin + 1), key2 = key_behind(key1, begin + 2);
    load_page(key);

    // this lane's row
    const int row = wave * 32 + col, r = t.r0 + row, token = r / p.group, q_head = head * p.group + r % p.group;
    const bool live = row < t.rows;
    const int position = live ? t.start + token : -1;
    v8 q[CH][2];
#pragma unroll
    for (int ch = 0; ch < CH; ++ch)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            q[ch][j] = v8{};
            if (live) q[ch][j] = load_q<T>((const T*)p.q + (int64_t)(t.first + token) * p.q_row + (int64_t)q_head * p.q_head + ch * 32 + h * 16 + j * 8, p.scale_log2 < 0.f);
        }
    // the first 32 keys from `none` on are seen by no row of the wave; those at `last_whole` and before, and behind `first_whole`, by all
    const int wave_rows = min(t.rows - wave * 32, 32);
    const int none = wave_rows > 0 ? t.start + (t.r0 + wave * 32 + wave_rows - 1) / p.group + 1 : 0;
    const int last_whole = t.start + (t.r0 + wave * 32) / p.group - 31, first_whole = p.window ? none - 1 - p.window : -1;
    if (begin < end) {
        load_codes(key, 0);
        load_page(key1);
    }
    v16f o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = v16f{};
    float m = live ? kMinusInf : 0.f, l = 0.f;
    ValueScale<T> value;
    const int s_key = 16 * ((col >> 2) & 1) + 4 * (col >> 3) + (col & 3);  // the key that this lane reads as a row of K, of 32
    const int k_lane = s_key * D + (h ^ k_swizzle<D>(s_key)) * 16, v_lane = col * 64 + (h ^ v_swizzle(col)) * 16;
    for (int step = begin; step < end; ++step, key = key1, key1 = key2) {
        const int buffer = (step - begin) & 1;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();  // this step's codes are there for all, and all are done with the other buffer
        float factor[HALVES], this_v_scale[HALVES];
        bool page_there[HALVES];
#pragma unroll
        for (int i = 0; i < HALVES; ++i) factor[i] = score_factor(k_scale[i], p.scale_log2), this_v_scale[i] = v_scale[i], page_there[i] = there[i].there;
        key2 = key_behind(key1, step + 2);
        if (step + 1 < end) {
            load_codes(key1, buffer ^ 1);
            load_page(key2);
        }
        if (key >= none) continue;
        // (with ONE, a scalar: whether any key of the step's page is seen by the tile)
        if constexpr (ONE) value.set(this_v_scale[0], page_there[0] && key < t.key1 && (key + 64 > t.key0 || key < p.sinks));
        // fragments are asked for a phase ahead (k's of the second half in front of the first half's second product, v's in front of
        // the softmax), pinned by fences: behind each other, a read's latency and its use would add up 16 times a step
        // (the chunks of a fragment's rows differ from the first one's in an exclusive or of their number, which the swizzle leaves alone)
        v4i kc[CH], vc[DT];
        const int k_first = k_lane + buffer * (64 * D), v_first = v_lane + buffer * (64 * D);
        auto read_k = [&](int half) {
#pragma unroll
            for (int ch = 0; ch < CH; ++ch) kc[ch] = *reinterpret_cast<const v4i*>(&lds_k[0][0] + (k_first ^ (ch * 32)) + half * 32 * D);
            if constexpr (D < 256) __builtin_amdgcn_sched_barrier(0);
        };
        read_k(0);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int key_h = key + 32 * half, first = key_h + 16 * h, i_h = ONE ? 0 : half;
            if (half == 1 && key_h >= none) continue;
            Scores32 s;
            s.x = v16f{};
#pragma unroll
            for (int ch = 0; ch < CH; ++ch) {
                s.x = mfma32(widen<T>(kc[ch][0], kc[ch][1]), q[ch][0], s.x);
                s.x = mfma32(widen<T>(kc[ch][2], kc[ch][3]), q[ch][1], s.x);
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                vc[d] = *reinterpret_cast<const v4i*>(&lds_v[0][0] + (v_first ^ (half * 32)) + d * 32 * 64);
            }
            if constexpr (D < 256) __builtin_amdgcn_sched_barrier(0);
            bool whole = key_h <= last_whole && key_h > first_whole;
            if constexpr (ONE) {
                whole = whole && page_there[0];
            } else {
                whole = whole && __ballot(!page_there[i_h]) == 0;
                value.set(this_v_scale[i_h], whole || (page_there[i_h] && first < t.key1 && (first + 16 > t.key0 || first < p.sinks)));
            }
            if (!whole) {
                asm volatile("");  // (keeps the selection a branch)
                select_seen(s, first, position, p.window, p.sinks, page_there[i_h]);
#pragma unroll
                for (int d = 0; d < DT; ++d) vc[d] = seen_codes(vc[d], t, p.sinks, first, page_there[i_h]);
            }
            v8 pt[2];
            const float rescale = weigh<T>(s, factor[i_h], value, m, l, pt);
            if (__ballot(rescale != 1.f)) {
#pragma unroll
                for (int d = 0; d < DT; ++d) o[d] *= rescale;
            }
            if (half == 0) read_k(1);
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                o[d] = mfma32(widen<T>(vc[d][0], vc[d][1]), pt[0], o[d]);
                o[d] = mfma32(widen<T>(vc[d][2], vc[d][3]), pt[1], o[d]);
            }
        }
    }

    const float sum = l + __shfl_xor(l, 32);
    int last = t.r0 + row;
    asm("" : "+v"(last));  // (worked out again, not held through the loop)
    if (row >= t.rows) return;
    const int64_t out_row = (int64_t)(t.first + last / p.group) * p.q_heads + head * p.group + last % p.group;
    if (p.splits > 1) {
        const int64_t at = (int64_t)split * c.rows * p.q_heads + out_row;
        if (h == 0) p.part_ml[2 * at] = m, p.part_ml[2 * at + 1] = sum;
        if (!(sum == 0.f)) {
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int a = 0; a < 4; ++a)
                    *reinterpret_cast<v4f*>(p.part_o + at * D + d * 32 + 8 * a + 4 * h) = v4f{o[d][4 * a], o[d][4 * a + 1], o[d][4 * a + 2], o[d][4 * a + 3]} * ValueScale<T>::kDown;
        }
    } else {
        typedef T v4t __attribute__((ext_vector_type(4)));
        const float f = sum == 0.f ? 0.f : ValueScale<T>::kDown / sum;  // a row that sees nothing is zero
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                const v4f x = v4f{o[d][4 * a], o[d][4 * a + 1], o[d][4 * a + 2], o[d][4 * a + 3]} * f;
                *reinterpret_cast<v4t*>((T*)p.out + out_row * D + d * 32 + 8 * a + 4 * h) = __builtin_convertvector(x, v4t);
            }
    }
}

// out = sum over splits of exp2(m_s - m) O_s, over the sum of exp2(m_s - m) l_s, in the order of the splits: D / 4 lanes per row of q.  All
// splits' m and l, and the first four parts of O, are asked for at once; then O, four in flight.  Parts with no weight were not written.  Empty is what has a sum of
// zero and nothing else: a sum that is no number (NaN in q, a score that overflowed) makes the row's sum, and so the row, no number.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv_attention_join_kernel(const KvAttentionParams p) {
    constexpr int QUADS = D / 4, ROWS = 256 / QUADS;
    __shared__ float weight[ROWS][kMostSplits];
    const int tid = (int)threadIdx.x, lane = tid % QUADS;
    const int64_t rows = (int64_t)p.c.rows * p.q_heads, row = (int64_t)blockIdx.x * ROWS + tid / QUADS;
    const int token = (int)(min(row, rows - 1) / p.q_heads);
    // rows of no sequence are left as they were
    const bool live = row < rows && token >= clamp_row(p.c.indptr[0], p.c.rows) && token < clamp_row(p.c.indptr[p.c.batch], p.c.rows);
    const float* part_at = p.part_o + row * D + 4 * lane;
    const int64_t part_step = rows * D;
    v4f part[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        part[i] = v4f{0.f, 0.f, 0.f, 0.f};
        if (live && i < p.splits) part[i] = *reinterpret_cast<const v4f*>(part_at + i * part_step);
    }
    constexpr int EACH = kMostSplits / QUADS > 0 ? kMostSplits / QUADS : 1;
    float m[EACH], l[EACH], top = kMinusInf, sum = 0.f;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int s = lane + i * QUADS;
        m[i] = kMinusInf, l[i] = 0.f;
        if (live && s < p.splits) m[i] = p.part_ml[2 * (s * rows + row)], l[i] = p.part_ml[2 * (s * rows + row) + 1];
        top = fmaxf(top, m[i]);
    }
#pragma unroll
    for (int d = 1; d < QUADS; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
    const float base = top == kMinusInf ? 0.f : top;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const float f = l[i] == 0.f ? 0.f : __builtin_amdgcn_exp2f(m[i] - base);
        if (lane + i * QUADS < kMostSplits) weight[tid / QUADS][lane + i * QUADS] = f;
        sum += f * l[i];
    }
#pragma unroll
    for (int d = 1; d < QUADS; d <<= 1) sum += __shfl_xor(sum, d);
    __syncthreads();
    if (!live) return;
    v4f x = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < p.splits; s0 += 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float f = s0 + i < p.splits ? weight[tid / QUADS][s0 + i] : 0.f;
            if (f > 0.f) x += f * part[i];
            // the next four: a part without weight may hold anything and is left out by selection
            if (s0 + 4 + i < p.splits) part[i] = *reinterpret_cast<const v4f*>(part_at + (s0 + 4 + i) * part_step);
        }
    }
    typedef T v4t __attribute__((ext_vector_type(4)));
    x *= sum == 0.f ? 0.f : 1.0f / sum;
    *reinterpret_cast<v4t*>((T*)p.out + row * D + 4 * lane) = __builtin_convertvector(x, v4t);
}

// Tiles there can be: sum over sequences of ceil(n * group / tile_rows) at most.
int64_t row_tiles(const KvAttentionParams& p, int64_t tile_rows) { return (int64_t)p.c.rows * p.group / tile_rows + p.c.batch; }
// Rows that a sequence's key/value head has on average, and tiles of so many in all sequences and heads: the host does not read the tensors.
int64_t rows_each(const KvAttentionParams& p) { return ((int64_t)p.c.rows * p.group + p.c.batch - 1) / p.c.batch; }
int64_t attention_blocks(const KvAttentionParams& p, int64_t tile_rows) { return row_tiles(p, tile_rows) * p.c.heads * p.splits; }
int64_t join_blocks(const KvAttentionParams& p) { return ((int64_t)p.c.rows * p.q_heads * (p.c.dim / 4) + 255) / 256; }
int64_t tiles_in_all(const KvAttentionParams& p, int64_t tile_rows) { return p.c.batch * ((rows_each(p) + tile_rows - 1) / tile_rows) * p.c.heads; }

// Keys that a tile can see, as far as the host can tell.
int64_t keys_at_most(const KvAttentionParams& p) {
    const int64_t keys = (int64_t)p.c.width << p.c.page_log2;
    return p.window ? std::min<int64_t>(keys, (int64_t)p.window + 128 + ((int64_t)p.sinks + 63) / 64 * 64) : keys;
}

}  // namespace

// Rows of a tile: 16 or 32 in the form for few rows, 128 in the one for many.  A workgroup of the first runs through its steps fastest with 16 rows,
// but every tile reads the keys, and a compute unit holds one workgroup.  So (128 elements, 8 heads; us with tiles of 16 / 32 / 128 rows):
//   16 while the compute units hold all tiles, up to two a sequence, which share an XCD's cache if workgroups 8 apart have the same head (4
//   sequences of 20 rows and 3000 keys 14.6 / 18.0 / 23; 32 of 20 rows 48 / 38 / 44; 64 of 20 rows and 2 heads 35 / 27 / 32), and
//   more of them only up to a quarter of the compute units (1 of 64 rows 13.8 / 16.9 / 20.6; 8 of 80 rows and 8000 keys 96 / 54 / 64);
//   32 while the compute units hold all tiles (2 of 512 rows 45 / 27 / 39), or twice as many if the keys are read twice at most and not so few that the
//   workgroups' beginnings and ends count (32 of 48 rows: 3000 keys 67 / 53 / 65, 500 keys 29 / 26 / 18; 16 of 96 rows 67 / 51 / 46);
//   of 256 elements there is no form of 32 rows, and 128 of them take all registers, one wave per SIMD: 16 up to 32 rows each (64 of 20 rows 185 / - / 254) and
//   up to twice the compute units (16 of 48 rows 80 / - / 105, of 96 rows 120 / - / 85).
int kv_attention_tile_rows(const KvAttentionParams& p) {
    const int64_t each = rows_each(p), by16 = tiles_in_all(p, 16), by32 = tiles_in_all(p, 32);
    if (each <= 16 || by16 <= (each <= 32 && p.c.heads % 8 == 0 ? kComputeUnits : kComputeUnits / 4)) return 16;
    if (p.c.dim == 256) return each <= 32 || by16 <= 2 * kComputeUnits ? 16 : 128;
    if (by32 <= kComputeUnits) return 32;
    return keys_at_most(p) > 1024 && (each <= 32 || (each <= 64 && by32 <= 2 * kComputeUnits)) ? 32 : 128;
}

namespace {

template <typename T, int D>
hipError_t launch(KvAttentionParams p, hipStream_t s) {
    const int tile_rows = kv_attention_tile_rows(p);
    const int64_t blocks = attention_blocks(p, tile_rows);
    const dim3 grid((unsigned)blocks), block(256);
    // more workgroups than compute units, whole sequences each: the long ones first, and the short ones fill in behind them (64 sequences of 100
    // to 8000 keys 98 us, in their own order 110; 40 of them 74 and 83; of 4000 each 101 and 100)
    p.longest_first = tile_rows == 16 && p.splits == 1 && p.c.batch <= 64 && p.c.batch > 1 && blocks > kComputeUnits;
    const bool one = p.c.page_log2 >= 6;
#define TG_FEW(NT, ONE) hipLaunchKernelGGL((kv_attention_kernel<T, D, NT, ONE>), grid, dim3(64 * kFewWaves<D>), 0, s, p)
    if (tile_rows == 128) {
        if (one) hipLaunchKernelGGL((kv_attention_rows_kernel<T, D, true>), grid, block, 0, s, p);
        else hipLaunchKernelGGL((kv_attention_rows_kernel<T, D, false>), grid, block, 0, s, p);
    } else if (tile_rows == 16) {
        if (one) TG_FEW(1, true);
        else TG_FEW(1, false);
    } else if constexpr (D != 256) {
        if (one) TG_FEW(2, true);
        else TG_FEW(2, false);
    }
#undef TG_FEW
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits == 1) return e;
    hipLaunchKernelGGL((kv_attention_join_kernel<T, D>), dim3((unsigned)join_blocks(p)), block, 0, s, p);
    return hipGetLastError();
}

}  // namespace

int kv_attention_splits(const KvAttentionParams& p) {
    const int tile_rows = kv_attention_tile_rows(p);
    // Few rows: tiles as far as the host can tell, and a workgroup per compute unit (of 128 elements, two do not fit its registers), never
    // more: 12 sequences of 4000 keys x 8 heads 23.4 us cut in two, 32.5 cut in three (288 workgroups); 20 such uncut 29.6, cut in two 41.2;
    // 8 of 8000 cut in four 27.6, uncut 48.6.  Shares of one size for long and short sequences, counted on the device, were no faster: the
    // memory is shared by those that still run.  Many rows: two workgroups per compute unit.  No share below 8 steps, and none up to 1024 keys
    // (8 x 1000 keys 11.5 us in one launch, 12.0 cut and joined).
    const int64_t units = tile_rows != 128 ? tiles_in_all(p, tile_rows) : row_tiles(p, tile_rows) * p.c.heads;
    const int64_t steps = (keys_at_most(p) + 63) / 64, workgroups = tile_rows != 128 ? kComputeUnits : 2 * kComputeUnits;
    const int64_t wanted = tile_rows != 128 ? workgroups / units : (workgroups + units / 2) / units, most = steps <= 2 * kLeastSteps ? 1 : (steps + kLeastSteps - 1) / kLeastSteps;
    return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(wanted, most), kMostSplits));
}

int64_t kv_attention_threads(const KvAttentionParams& p) {
    const int tile_rows = kv_attention_tile_rows(p), waves = tile_rows == 128 ? 4 : p.c.dim == 256 ? kFewWaves<256> : kFewWaves<128>;
    return std::max(attention_blocks(p, tile_rows) * 64 * waves, p.splits > 1 ? join_blocks(p) * 256 : 0);
}

hipError_t run_kv_attention(const KvAttentionParams& p, bool is_bf16, hipStream_t s) {
    if (p.c.rows <= 0 || p.c.batch <= 0) return hipSuccess;
    switch (p.c.dim) {
        case 64: return is_bf16 ? launch<__bf16, 64>(p, s) : launch<_Float16, 64>(p, s);
        case 128: return is_bf16 ? launch<__bf16, 128>(p, s) : launch<_Float16, 128>(p, s);
        case 256: return is_bf16 ? launch<__bf16, 256>(p, s) : launch<_Float16, 256>(p, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace tg
