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
// Codes become the 16-bit type of q exactly (e4m3 has 4 significant bits).  k's scale joins the softmax's factor.  v's scale: O is
// held in units of the largest one seen, u; P is multiplied by v_scale / u <= 1 before it is rounded to 16 bits (2^-9 relative in
// bf16, 2^-12 in f16, of its own value), where a page differs from that.  S, m, l and O are fp32.
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

template <typename T> struct Types;
template <> struct Types<__bf16> { typedef bf16x8 v8; typedef bf16x2 v2; };
template <> struct Types<_Float16> { typedef f16x8 v8; typedef f16x2 v2; };

__device__ __forceinline__ v4f mfma16(bf16x8 a, bf16x8 b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ v4f mfma16(f16x8 a, f16x8 b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

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

constexpr float kMinusInf = -__builtin_inff();
constexpr float kSmallestUnit = 0x1p-126f;
// The maximum that scores are taken against moves only when it has grown by more than this (in powers of two): weights are then at most
// 2^8, which costs no precision in floating point, and O is rescaled a few times in all instead of in most steps.
constexpr float kSlack = 8.f;

// The rows of one workgroup and the steps of 64 keys that any of them sees.
struct RowTile {
    int seq, head;          // sequence, key/value head
    int first, r0, rows;    // sequence's first packed row; the tile's first row of the sequence, and how many it has
    int64_t start;          // position of the sequence's first new token
    int64_t low, high;      // positions of the tile's first and last row
    int64_t key0, key1;     // keys [key0, key1) and, below key0, [0, sinks)
    int steps, sink_steps;  // steps of 64 keys: sink_steps from 0 on, then from key0 / 64 on
    __device__ __forceinline__ int64_t key_of(int step) const { return step < sink_steps ? (int64_t)step * 64 : ((key0 >> 6) + step - sink_steps) * 64; }
};

__device__ __forceinline__ bool find_tile(const KvAttentionParams& p, int tile_rows, int item, int head, RowTile& t) {
    const KvCache& c = p.c;
    const SeqItem f = find_sequence(c.indptr, c.batch, c.rows, item, p.group, tile_rows, 1);
    if (f.seq < 0) return false;
    const int64_t r0 = (int64_t)f.item * tile_rows, total = (int64_t)f.n * p.group;
    if (r0 >= total) return false;
    t.seq = f.seq, t.head = head, t.first = f.first;
    t.r0 = (int)r0, t.rows = (int)min((int64_t)tile_rows, total - r0);
    t.start = (int64_t)max(c.lens[f.seq], 0) - f.n;
    t.low = t.start + t.r0 / p.group, t.high = t.start + (t.r0 + t.rows - 1) / p.group;
    const int64_t capacity = (int64_t)c.width << c.page_log2;
    t.key1 = max(min(t.high + 1, capacity), (int64_t)0);
    t.key0 = p.window ? min(max(t.low - p.window + 1, (int64_t)0), t.key1) : 0;
    const int64_t sinks = min((int64_t)p.sinks, t.key0);
    t.sink_steps = (int)min((sinks + 63) >> 6, t.key0 >> 6);
    t.steps = t.key1 > 0 ? t.sink_steps + (int)(((t.key1 + 63) >> 6) - (t.key0 >> 6)) : 0;
    return true;
}

// A page for lane's 16 keys from `key` on, or one that may be read in its place (its keys are then not seen).
struct Granule {
    int page;
    bool there;
};
__device__ __forceinline__ Granule granule_of(const KvCache& c, int seq, int64_t key) {
    const int64_t index = min(key >> c.page_log2, (int64_t)c.width - 1);
    const int page = c.table[(int64_t)seq * c.width + index];
    Granule g;
    g.there = page >= 0 && page < c.pages;
    g.page = g.there ? page : 0;
    return g;
}

// Four waves, 16 rows; the waves take the steps of the workgroup's share in turn and join at the end.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv_attention_kernel(const KvAttentionParams p) {
    typedef typename Types<T>::v8 v8;
    constexpr int CH = D / 64, DT = D / 16;  // 64-element chunks of a key, 16-element tiles of a value
    const KvCache& c = p.c;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, g = lane >> 4;
    const int split = (int)blockIdx.x % p.splits, rest = (int)blockIdx.x / p.splits;
    RowTile t;
    if (!find_tile(p, 16, rest / c.heads, rest % c.heads, t)) return;
    const int share = max((t.steps + p.splits - 1) / p.splits, 4);
    const int begin = min(split * share, t.steps), end = min(begin + share, t.steps);

    // this lane's row
    const int r = t.r0 + col, token = r / p.group, q_head = t.head * p.group + r % p.group;
    const bool row_live = col < t.rows;
    const int64_t position = row_live ? t.start + token : -1;
    v8 q[CH][2];
#pragma unroll
    for (int ch = 0; ch < CH; ++ch)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (row_live) q[ch][h] = *reinterpret_cast<const v8*>((const T*)p.q + (int64_t)(t.first + token) * p.q_row + (int64_t)q_head * p.q_head + ch * 64 + g * 16 + h * 8);
            else q[ch][h] = v8{};
        }

    const int P = 1 << c.page_log2, in_page = P - 1;
    const int64_t block_bytes = (int64_t)P * D;
    v4f o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = v4f{0.f, 0.f, 0.f, 0.f};
    float m = kMinusInf, l = 0.f, u = kSmallestUnit;

    for (int step = begin + wave; step < end; step += 4) {
        const int64_t key = t.key_of(step);
        const int64_t mine = key + 16 * g;  // this lane's 16 keys, as columns of V^T
        const Granule kg = granule_of(c, t.seq, key + 16 * (col >> 2)), vg = granule_of(c, t.seq, mine);
        const uint8_t* kp = c.k + ((int64_t)kg.page * c.heads + t.head) * block_bytes + (int64_t)((key + 16 * (col >> 2) + (col & 3)) & in_page) * D + g * 16;
        const uint8_t* vp = c.v + ((int64_t)vg.page * c.heads + t.head) * block_bytes + col * P + (mine & in_page);
        v4i kc[4][CH], vc[DT];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int ch = 0; ch < CH; ++ch) kc[i][ch] = *reinterpret_cast<const v4i*>(kp + i * 4 * D + ch * 64);
#pragma unroll
        for (int d = 0; d < DT; ++d) vc[d] = *reinterpret_cast<const v4i*>(vp + d * 16 * P);
        const int64_t at = (int64_t)vg.page * c.heads + t.head;
        const float k_scale = c.k_scale[at];
        float v_scale = c.v_scale[at];

        v4f s[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[i] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ch = 0; ch < CH; ++ch) {
                s[i] = mfma16(widen<T>(kc[i][ch][0], kc[i][ch][1]), q[ch][0], s[i]);
                s[i] = mfma16(widen<T>(kc[i][ch][2], kc[i][ch][3]), q[ch][1], s[i]);
            }
        }
        const float factor = k_scale * p.scale_log2;
        // every key of the step seen by every row: nothing to select
        const bool whole = key + 63 <= t.low && (!p.window || key > t.high - p.window) && __ballot(!vg.there) == 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] *= factor;
        if (!whole) {
            const int64_t first_seen = p.window ? position - p.window + 1 : 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int64_t j = mine + i;
                const bool seen = vg.there && j <= position && (j >= first_seen || j < p.sinks);
                s[i / 4][i % 4] = seen ? s[i / 4][i % 4] : kMinusInf;
            }
            // codes that no row sees: behind the last key, before the window, in no page
            const bool any = vg.there && mine < t.key1 && (mine + 16 > t.key0 || mine < p.sinks);
            const int live = any ? (int)min(t.key1 - mine, (int64_t)16) : 0;
            if (!any) v_scale = 0.f;
            v4i mask;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int bytes = min(max(live - 4 * w, 0), 4);
                mask[w] = bytes == 4 ? -1 : (1 << (8 * bytes)) - 1;
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) vc[d] &= mask;
        }
        float top = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3]));
#pragma unroll
        for (int i = 1; i < 4; ++i) top = fmaxf(top, fmaxf(fmaxf(s[i][0], s[i][1]), fmaxf(s[i][2], s[i][3])));
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float m_new = fmaxf(m, top), base = m_new == kMinusInf ? 0.f : m_new;
        const float shrink = __builtin_amdgcn_exp2f(m - base);
        float unit = fmaxf(v_scale, __shfl_xor(v_scale, 16));
        unit = fmaxf(fmaxf(unit, __shfl_xor(unit, 32)), u);
        const float ratio = v_scale / unit, rescale = shrink * (u / unit);
        m = m_new, u = unit;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[i][j] = __builtin_amdgcn_exp2f(s[i][j] - base);
                sum += s[i][j];
                s[i][j] *= ratio;
            }
        l = l * shrink + sum;
        typename Types<T>::v8 pt[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
            pt[h] = __builtin_convertvector(__builtin_shufflevector(s[2 * h], s[2 * h + 1], 0, 1, 2, 3, 4, 5, 6, 7), v8);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            o[d] *= rescale;
            o[d] = mfma16(widen<T>(vc[d][0], vc[d][1]), pt[0], o[d]);
            o[d] = mfma16(widen<T>(vc[d][2], vc[d][3]), pt[1], o[d]);
        }
    }

    // the four waves' results: m, l and u, then O, each in units of the largest
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    __shared__ float part_m[4][16], part_l[4][16], part_u[4];
    __shared__ float part_o[4][16][D + 4];
    if (lane < 16) part_m[wave][col] = m, part_l[wave][col] = l;
    if (lane == 0) part_u[wave] = u;
    __syncthreads();
    float top = part_m[0][col], unit = part_u[0];
#pragma unroll
    for (int w = 1; w < 4; ++w) top = fmaxf(top, part_m[w][col]), unit = fmaxf(unit, part_u[w]);
    const float base = top == kMinusInf ? 0.f : top, mine = __builtin_amdgcn_exp2f(m - base) * (u / unit);
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<v4f*>(&part_o[wave][col][d * 16 + 4 * g]) = o[d] * mine;
    __syncthreads();
    constexpr int QUADS = D / 4;
    for (int i = tid; i < t.rows * QUADS; i += 256) {
        const int row = i / QUADS, e = 4 * (i % QUADS), rr = t.r0 + row;
        float row_top = part_m[0][row];
#pragma unroll
        for (int w = 1; w < 4; ++w) row_top = fmaxf(row_top, part_m[w][row]);
        const float row_base = row_top == kMinusInf ? 0.f : row_top;
        float sum = 0.f;
        v4f x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            sum += part_l[w][row] * __builtin_amdgcn_exp2f(part_m[w][row] - row_base);
            x += *reinterpret_cast<const v4f*>(&part_o[w][row][e]);
        }
        x *= unit;
        const int64_t out_row = (int64_t)(t.first + rr / p.group) * p.q_heads + t.head * p.group + rr % p.group;
        if (p.splits > 1) {
            const int64_t at = (int64_t)split * c.rows * p.q_heads + out_row;
            if (e == 0) p.part_ml[2 * at] = row_top, p.part_ml[2 * at + 1] = sum;
            if (sum > 0.f) *reinterpret_cast<v4f*>(p.part_o + at * D + e) = x;
        } else {
            typedef T v4t __attribute__((ext_vector_type(4)));
            x *= sum > 0.f ? 1.0f / sum : 0.f;  // a row that sees nothing is zero
            *reinterpret_cast<v4t*>((T*)p.out + out_row * D + e) = __builtin_convertvector(x, v4t);
        }
    }
}

// Many rows: 128 of them per workgroup, 32 per wave, and every wave runs over the same keys, whose codes are staged in LDS for all
// four: 16 bytes per lane and load through registers, the next step's while this one's products run, in two buffers with one
// barrier a step.  Codes stay e4m3 in LDS (half the reads that 16 bits would cost) and are widened behind each read for 32 rows.
// 16-byte chunks are placed so that the 16 lanes that read together (16 rows of one fragment, one chunk each) cover all banks:
//   k, chunks of row `key`: chunk ^ f, rows of a fragment being 16 a + 4 i + b;  v, 4 chunks a row: chunk ^ (row / 4) % 4
template <int D>
__device__ __forceinline__ int k_swizzle(int row) {
    const int a = (row >> 4) & 3, b = row & 3;
    return D == 64 ? a : D == 128 ? 2 * a + (b >> 1) : 4 * a + b;
}
__device__ __forceinline__ int v_swizzle(int row) { return (row >> 2) & 3; }

template <typename T, int D>
__global__ void __launch_bounds__(256, D == 256 ? 1 : 2) kv_attention_rows_kernel(const KvAttentionParams p, int items) {
    typedef typename Types<T>::v8 v8;
    constexpr int CH = D / 64, DT = D / 16, LOADS = D / 64, KCH = D / 16;
    __shared__ __align__(16) uint8_t lds_k[2][64 * D], lds_v[2][64 * D];
    const KvCache& c = p.c;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 15, g = lane >> 4;
    const int head = (int)blockIdx.x % c.heads, rest = (int)blockIdx.x / c.heads, split = rest % p.splits;
    RowTile t;
    if (!find_tile(p, 128, items - 1 - rest / p.splits, head, t)) return;  // (the last rows of a sequence, which see most, first)
    const int share = max((t.steps + p.splits - 1) / p.splits, 4);
    const int begin = min(split * share, t.steps), end = min(begin + share, t.steps);

    // this lane's two rows
    int64_t position[2];
    v8 q[2][CH][2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        const int row = wave * 32 + n * 16 + col, r = t.r0 + row, token = r / p.group, q_head = head * p.group + r % p.group;
        position[n] = row < t.rows ? t.start + token : -1;
#pragma unroll
        for (int ch = 0; ch < CH; ++ch)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (row < t.rows) q[n][ch][h] = *reinterpret_cast<const v8*>((const T*)p.q + (int64_t)(t.first + token) * p.q_row + (int64_t)q_head * p.q_head + ch * 64 + g * 16 + h * 8);
                else q[n][ch][h] = v8{};
            }
    }
    const int wave_rows = min(t.rows - wave * 32, 32);
    const int64_t wave_low = t.start + (t.r0 + wave * 32) / p.group, wave_high = t.start + (t.r0 + wave * 32 + wave_rows - 1) / p.group;

    const int P = 1 << c.page_log2, in_page = P - 1;
    const int64_t block_bytes = (int64_t)P * D;
    v4f o[2][DT];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int d = 0; d < DT; ++d) o[n][d] = v4f{0.f, 0.f, 0.f, 0.f};
    float m[2] = {kMinusInf, kMinusInf}, l[2] = {0.f, 0.f}, u = kSmallestUnit;

    // a step's pages, one per group of 16 lanes, then its codes and scales on their way to LDS
    v4i k_reg[LOADS], v_reg[LOADS];
    float k_scale, v_scale;
    Granule page{0, false}, there{0, false};
    auto load_page = [&](int step) { if (step < end) page = granule_of(c, t.seq, t.key_of(step) + 16 * g); };
    auto load_codes = [&](int step) {
        there = page;
        const int64_t key = t.key_of(step), at = (int64_t)page.page * c.heads + head;
        k_scale = c.k_scale[at], v_scale = c.v_scale[at];
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int ci = tid + 256 * j, row = ci / KCH, chunk = (ci % KCH) ^ k_swizzle<D>(row);
            const int64_t block = (int64_t)__shfl(page.page, (row >> 4) * 16) * c.heads + head;
            k_reg[j] = *reinterpret_cast<const v4i*>(c.k + block * block_bytes + (int64_t)((key + row) & in_page) * D + chunk * 16);
        }
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int ci = tid + 256 * j, row = ci / 4, chunk = (ci & 3) ^ v_swizzle(row);
            const int64_t block = (int64_t)__shfl(page.page, chunk * 16) * c.heads + head;
            v_reg[j] = *reinterpret_cast<const v4i*>(c.v + block * block_bytes + (int64_t)row * P + ((key + 16 * chunk) & in_page));
        }
    };
    auto store_codes = [&](int step, int buffer) {
        const int64_t key = t.key_of(step);
        const bool whole = key + 64 <= t.key1 && key >= t.key0 && __ballot(!there.there) == 0;
#pragma unroll
        for (int j = 0; j < LOADS; ++j) *reinterpret_cast<v4i*>(&lds_k[buffer][(tid + 256 * j) * 16]) = k_reg[j];
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int ci = tid + 256 * j, chunk = (ci & 3) ^ v_swizzle(ci / 4);
            if (!whole) {  // codes that no row sees: behind the last key, before the window, in no page
                const int64_t first = key + 16 * chunk;
                const bool any = __shfl((int)there.there, chunk * 16) && first < t.key1 && (first + 16 > t.key0 || first < p.sinks);
                const int live = any ? (int)min(t.key1 - first, (int64_t)16) : 0;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const int bytes = min(max(live - 4 * w, 0), 4);
                    v_reg[j][w] &= bytes == 4 ? -1 : (1 << (8 * bytes)) - 1;
                }
            }
            *reinterpret_cast<v4i*>(&lds_v[buffer][ci * 16]) = v_reg[j];
        }
    };

    if (begin < end) {
        load_page(begin);
        load_codes(begin);
        load_page(begin + 1);
        store_codes(begin, 0);
    }
    __syncthreads();
    for (int step = begin; step < end; ++step) {
        const int buffer = (step - begin) & 1;
        const int64_t key = t.key_of(step), mine = key + 16 * g;
        const float factor = k_scale * p.scale_log2;
        float v_unit = v_scale;
        const bool page_there = there.there;
        if (step + 1 < end) {
            load_codes(step + 1);
            load_page(step + 2);
        }
        if (wave_rows > 0 && key <= wave_high) {
            v4f s[2][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[0][i] = s[1][i] = v4f{0.f, 0.f, 0.f, 0.f};
                const int row = 16 * (col >> 2) + 4 * i + (col & 3);
#pragma unroll
                for (int ch = 0; ch < CH; ++ch) {
                    const v4i kc = *reinterpret_cast<const v4i*>(&lds_k[buffer][row * D + ((ch * 4 + g) ^ k_swizzle<D>(row)) * 16]);
                    const v8 a = widen<T>(kc[0], kc[1]), b = widen<T>(kc[2], kc[3]);
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        s[n][i] = mfma16(a, q[n][ch][0], s[n][i]);
                        s[n][i] = mfma16(b, q[n][ch][1], s[n][i]);
                    }
                }
            }
            const bool whole = key + 63 <= wave_low && (!p.window || key > wave_high - p.window) && __ballot(!page_there) == 0;
            if (!whole && !(page_there && mine < t.key1 && (mine + 16 > t.key0 || mine < p.sinks))) v_unit = 0.f;
            float unit = fmaxf(v_unit, __shfl_xor(v_unit, 16));
            unit = fmaxf(fmaxf(unit, __shfl_xor(unit, 32)), u);
            const float ratio = v_unit / unit;
            float rescale[2];
            v8 pt[2][2];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
#pragma unroll
                for (int i = 0; i < 4; ++i) s[n][i] *= factor;
                if (!whole) {
                    const int64_t first_seen = p.window ? position[n] - p.window + 1 : 0;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int64_t j = mine + i;
                        const bool seen = page_there && j <= position[n] && (j >= first_seen || j < p.sinks);
                        s[n][i / 4][i % 4] = seen ? s[n][i / 4][i % 4] : kMinusInf;
                    }
                }
                float top = fmaxf(fmaxf(s[n][0][0], s[n][0][1]), fmaxf(s[n][0][2], s[n][0][3]));
#pragma unroll
                for (int i = 1; i < 4; ++i) top = fmaxf(top, fmaxf(fmaxf(s[n][i][0], s[n][i][1]), fmaxf(s[n][i][2], s[n][i][3])));
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                const float m_new = top > m[n] + kSlack ? top : m[n], base = m_new == kMinusInf ? 0.f : m_new;
                const float shrink = __builtin_amdgcn_exp2f(m[n] - base);
                rescale[n] = m_new == m[n] ? u / unit : shrink * (u / unit);
                l[n] = m_new == m[n] ? l[n] : l[n] * shrink;
                m[n] = m_new;
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        s[n][i][j] = __builtin_amdgcn_exp2f(s[n][i][j] - base);
                        sum += s[n][i][j];
                    }
                l[n] += sum;
                if (__ballot(ratio != 1.f)) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[n][i] *= ratio;
                }
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    pt[n][h] = __builtin_convertvector(__builtin_shufflevector(s[n][2 * h], s[n][2 * h + 1], 0, 1, 2, 3, 4, 5, 6, 7), v8);
            }
            u = unit;
            if (__ballot(rescale[0] != 1.f || rescale[1] != 1.f)) {
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int d = 0; d < DT; ++d) o[n][d] *= rescale[n];
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const int row = d * 16 + col;
                const v4i vc = *reinterpret_cast<const v4i*>(&lds_v[buffer][row * 64 + (g ^ v_swizzle(row)) * 16]);
                const v8 a = widen<T>(vc[0], vc[1]), b = widen<T>(vc[2], vc[3]);
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    o[n][d] = mfma16(a, pt[n][0], o[n][d]);
                    o[n][d] = mfma16(b, pt[n][1], o[n][d]);
                }
            }
        }
        if (step + 1 < end) store_codes(step + 1, buffer ^ 1);
        __syncthreads();
    }

#pragma unroll
    for (int n = 0; n < 2; ++n) {
        float sum = l[n] + __shfl_xor(l[n], 16);
        sum += __shfl_xor(sum, 32);
        const int row = wave * 32 + n * 16 + col, r = t.r0 + row;
        if (row >= t.rows) continue;
        const int64_t out_row = (int64_t)(t.first + r / p.group) * p.q_heads + head * p.group + r % p.group;
        if (p.splits > 1) {
            const int64_t at = (int64_t)split * c.rows * p.q_heads + out_row;
            if (g == 0) p.part_ml[2 * at] = m[n], p.part_ml[2 * at + 1] = sum;
            if (sum > 0.f) {
#pragma unroll
                for (int d = 0; d < DT; ++d) *reinterpret_cast<v4f*>(p.part_o + at * D + d * 16 + 4 * g) = o[n][d] * u;
            }
        } else {
            typedef T v4t __attribute__((ext_vector_type(4)));
            const float f = sum > 0.f ? u / sum : 0.f;  // a row that sees nothing is zero
#pragma unroll
            for (int d = 0; d < DT; ++d) *reinterpret_cast<v4t*>((T*)p.out + out_row * D + d * 16 + 4 * g) = __builtin_convertvector(o[n][d] * f, v4t);
        }
    }
}

// out = sum over splits of exp2(m_s - m) O_s, over the sum of exp2(m_s - m) l_s: D / 4 lanes per row of q, in the order of the splits.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv_attention_join_kernel(const KvAttentionParams p) {
    constexpr int QUADS = D / 4;
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, rows = (int64_t)p.c.rows * p.q_heads, row = at / QUADS;
    if (row >= rows) return;
    // rows of no sequence are left as they were
    const int token = (int)(row / p.q_heads), e = 4 * (int)(at % QUADS);
    if (token < clamp_row(p.c.indptr[0], p.c.rows) || token >= clamp_row(p.c.indptr[p.c.batch], p.c.rows)) return;
    float top = kMinusInf;
    for (int s = 0; s < p.splits; ++s) top = fmaxf(top, p.part_ml[2 * (s * rows + row)]);
    const float base = top == kMinusInf ? 0.f : top;
    float sum = 0.f;
    v4f x = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < p.splits; ++s) {
        const float l = p.part_ml[2 * (s * rows + row) + 1];
        if (l > 0.f) {
            const float f = __builtin_amdgcn_exp2f(p.part_ml[2 * (s * rows + row)] - base);
            sum += f * l;
            x += f * *reinterpret_cast<const v4f*>(p.part_o + (s * rows + row) * D + e);
        }
    }
    typedef T v4t __attribute__((ext_vector_type(4)));
    x *= sum > 0.f ? 1.0f / sum : 0.f;
    *reinterpret_cast<v4t*>((T*)p.out + row * D + e) = __builtin_convertvector(x, v4t);
}

// Tiles that can begin: sum over sequences of ceil(n * group / tile_rows), see find_sequence.
int64_t row_tiles(const KvAttentionParams& p, int64_t tile_rows) { return (int64_t)p.c.rows * p.group / tile_rows + p.c.batch; }
// The form for many rows: by the rows that a sequence's key/value head has on average, as the host does not read the tensors.
bool many_rows(const KvAttentionParams& p) { return (int64_t)p.c.rows * p.group > 32 * (int64_t)p.c.batch; }

template <typename T, int D>
hipError_t launch(const KvAttentionParams& p, hipStream_t s) {
    const int64_t tile_rows = many_rows(p) ? 128 : 16, tiles = row_tiles(p, tile_rows), blocks = tiles * p.c.heads * p.splits;
    const int64_t join = ((int64_t)p.c.rows * p.q_heads * (D / 4) + 255) / 256;
    if (blocks > INT32_MAX || join > INT32_MAX) return hipErrorInvalidValue;
    if (many_rows(p)) hipLaunchKernelGGL((kv_attention_rows_kernel<T, D>), dim3((unsigned)blocks), dim3(256), 0, s, p, (int)tiles);
    else hipLaunchKernelGGL((kv_attention_kernel<T, D>), dim3((unsigned)blocks), dim3(256), 0, s, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits == 1) return e;
    hipLaunchKernelGGL((kv_attention_join_kernel<T, D>), dim3((unsigned)join), dim3(256), 0, s, p);
    return hipGetLastError();
}

}  // namespace

int kv_attention_splits(const KvAttentionParams& p) {
    const int64_t units = row_tiles(p, many_rows(p) ? 128 : 16) * p.c.heads;
    int64_t keys = (int64_t)p.c.width << p.c.page_log2;
    if (p.window) keys = std::min<int64_t>(keys, (int64_t)p.window + 128 + (p.sinks + 63) / 64 * 64);
    const int64_t steps = (keys + 63) / 64;
    const int64_t wanted = (512 + units - 1) / units, most = (steps + 3) / 4;
    return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(wanted, most), 64));
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
