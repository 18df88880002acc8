// Writing and reading the paged e4m3 cache (kv_device.h).
//
// Writing: rotary positions on the new tokens' q and k, then k and v in e4m3 with one scale per page and head.
//   rotary: pairs (a, b) of the first R elements of a head, (x[i], x[i + R/2]) or (x[2i], x[2i + 1]), turn by the table's angle of
//           the token's position: (a cos - b sin, a sin + b cos).  In fp32; k goes to e4m3 without a 16-bit rounding between.
//   scale:  2^e with the smallest e in [-40, 40] that brings the page's largest magnitude within 448.  e4m3 is a floating-point type: a
//           power of two costs its codes no precision, and moving stored codes from one power of two to a larger one only shifts their
//           exponents, exact but for e4m3's subnormals.  So a page that fills token by token keeps max(old, new) as its scale,
//           and its earlier codes move when the scale does: no token is rounded at more than one precision.
// One workgroup, or wave, writes the new tokens of one page, head and half of the cache: it alone reads and writes that scale, so no
// atomics, and the result does not depend on any order.  Bound by HBM at many tokens, by the launch and one chain
// of dependent loads (sequence, page, scale) at few, and by the moving of earlier codes where a page's scale grows.
#include <algorithm>

#include "kv_device.h"
#include "quant_device.h"

namespace tg {
namespace {

constexpr int kMinExponent = -40, kMaxExponent = 40;

// 2^e, the smallest with amax <= 448 * 2^e (448 = 1.75 * 2^8), from amax's bits
__device__ __forceinline__ float page_scale(float amax) {
    const uint32_t bits = __float_as_uint(amax);
    const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return __uint_as_float((uint32_t)(min(max(e, kMinExponent), kMaxExponent) + 127) << 23);
}

__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d) {
    int w = 0;  // (NaN: -448, as in the activation quantizer; a NaN code in v would reach rows that do not see its token)
    w = __builtin_amdgcn_cvt_pk_fp8_f32(__builtin_amdgcn_fmed3f(a, -448.f, 448.f), __builtin_amdgcn_fmed3f(b, -448.f, 448.f), w, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(__builtin_amdgcn_fmed3f(c, -448.f, 448.f), __builtin_amdgcn_fmed3f(d, -448.f, 448.f), w, true);
    return (uint32_t)w;
}

// Elements 8 c .. 8 c + 7 of a head (x: its first element), turned by table row `row` (cos, then sin; rotary % 16 == 0).
template <typename T>
__device__ __forceinline__ v8f_q load_turned(const T* x, int c, const float* row, int rotary, int interleaved) {
    v8f_q v = load8<T>(x + 8 * c);
    if (8 * c >= rotary) return v;  // (rotary 0: no rotation)
    const int half = rotary / 2;
    if (interleaved) {
        const v4f cs = *reinterpret_cast<const v4f*>(row + 4 * c), sn = *reinterpret_cast<const v4f*>(row + half + 4 * c);
        v8f_q y;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            y[2 * i] = v[2 * i] * cs[i] - v[2 * i + 1] * sn[i];
            y[2 * i + 1] = v[2 * i] * sn[i] + v[2 * i + 1] * cs[i];
        }
        return y;
    }
    const bool upper = 8 * c >= half;
    const int i0 = upper ? 8 * c - half : 8 * c;
    const v8f_q o = load8<T>(x + (upper ? 8 * c - half : 8 * c + half));  // the other member of each pair
    const v8f_q cs = load8<float>(row + i0), sn = load8<float>(row + half + i0);
    v8f_q y;
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = upper ? v[i] * cs[i] + o[i] * sn[i] : v[i] * cs[i] - o[i] * sn[i];
    return y;
}

// What lanes of one wave, or of the workgroup, have written to LDS is there for the others of them.
template <int WAVES>
__device__ __forceinline__ void lds_written() {
    if constexpr (WAVES > 1) {
        __syncthreads();
    } else {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
}

// Workgroups of the two kinds of work: first those that write the cache, then those that turn q.  A page, head and half is the work of WAVES
// waves: one where sequences have few new tokens (16 lanes of 8 elements have 128 of a token), else 4 or 16.
template <typename T, int WAVES>
__global__ void __launch_bounds__(64 * (WAVES > 4 ? WAVES : 4)) kv_append_kernel(const KvAppendParams p, int items, int cache_blocks, int v_pad, int q_waves) {
    constexpr int LANES = 64 * WAVES, BLOCK_WAVES = WAVES > 4 ? WAVES : 4;
    typedef T vecT __attribute__((ext_vector_type(8)));
    const KvCache& c = p.c;
    const int P = 1 << c.page_log2, D = c.dim, chunks = D / 8, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    if ((int)blockIdx.x >= cache_blocks) {
        // q: a wave has one token, and every q_waves-th 64 vectors of 8 elements of it
        const int64_t job = (int64_t)((int)blockIdx.x - cache_blocks) * BLOCK_WAVES + wave;
        // (the items are the rows that sequences have, in order; rows of no sequence are left as they were)
        if (job / q_waves >= c.rows) return;
        const SeqItem f = find_sequence(c, (int)(job / q_waves), [](int n, int) { return n; });
        if (f.seq < 0 || f.item >= f.n) return;
        const int64_t row = f.first + f.item, position = (int64_t)f.len - f.n + f.item;
        const float* angles = p.rope + min(max(position, (int64_t)0), (int64_t)p.rope_rows - 1) * p.rotary;
        const int vectors = p.q_heads * chunks;
        for (int i = (int)(job % q_waves) * 64 + ((int)threadIdx.x & 63); i < vectors; i += q_waves * 64) {
            const int head = i / chunks, ch = i - head * chunks;
            const v8f_q y = load_turned<T>((const T*)p.q + row * p.q_row + head * p.q_head, ch, angles, p.rotary, p.interleaved);
            *reinterpret_cast<vecT*>((T*)p.q_out + (row * p.q_heads + head) * D + 8 * ch) = __builtin_convertvector(y, vecT);
        }
        return;
    }
    extern __shared__ uint8_t all_lds[];  // v: the page's new codes, an element's tokens together, rows of v_pad bytes
    __shared__ float part[BLOCK_WAVES];
    const int unit = WAVES == 1 ? (int)blockIdx.x * 4 + wave : (int)blockIdx.x, tid = (int)threadIdx.x & (LANES - 1);
    uint8_t* lds = all_lds + (WAVES == 1 ? wave * D * v_pad : 0);
    const int half = unit & 1, head = (unit >> 1) % c.heads, item = (unit >> 1) / c.heads;
    if (item >= items) return;
    // pages from the one of the first new token's position (or of the sequence's beginning) to the last's
    const SeqItem f = find_sequence(c, item, [&](int n, int len) { return len > 0 ? ((len - 1) >> c.page_log2) - (max(len - n, 0) >> c.page_log2) + 1 : 0; });
    if (f.seq < 0) return;
    const int64_t len = f.len, start = len - f.n;  // position of the sequence's first new token
    const int64_t first = start > 0 ? start : 0, page_index = (first >> c.page_log2) + f.item;
    if (page_index >= c.width) return;
    const int64_t page_begin = page_index << c.page_log2;
    const int slot0 = (int)(first > page_begin ? first - page_begin : 0);
    const int slot1 = (int)min(len - page_begin, (int64_t)P);
    if (slot0 >= slot1) return;
    const int page = uniform_load(c.table + (int64_t)f.seq * c.width + page_index);
    if (page < 0 || page >= c.pages) return;
    const int64_t block = (int64_t)page * c.heads + head;
    float* scale_at = (half ? c.v_scale : c.k_scale) + block;
    uint8_t* codes = (half ? c.v : c.k) + block * ((int64_t)P * D);
    float old = 0.f;
    if (slot0 > 0) old = *scale_at;
    // rows of the packed input, and table rows, of the page's first slot on
    const int64_t row0 = f.first + (page_begin - start);
    const T* x = half ? (const T*)p.v + head * p.v_head : (const T*)p.k + head * p.k_head;
    const int64_t x_row = half ? p.v_row : p.k_row;
    const int rotary = half || !p.rope ? 0 : p.rotary;
    const int chunks_log2 = 31 - __clz(chunks), count = (slot1 - slot0) << chunks_log2;
    auto element = [&](int i) {
        const int slot = slot0 + (i >> chunks_log2), ch = i & (chunks - 1);
        const int64_t position = min(page_begin + slot, (int64_t)p.rope_rows - 1);
        return load_turned<T>(x + (row0 + slot) * x_row, ch, rotary ? p.rope + position * p.rotary : nullptr, rotary, p.interleaved);
    };
    // a lane's first vector stays in a register, the others are loaded again (held too, they cost more in waves per compute unit
    // than the second, cached, load: 4096 tokens 25 us, with two held 24.5 to 28, with four 33)
    v8f_q held = {};
    if (tid < count) held = element(tid);
    float amax = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) amax = fmaxf(amax, fabsf(held[k]));
    for (int i = tid + LANES; i < count; i += LANES) {
        const v8f_q v = element(i);
#pragma unroll
        for (int k = 0; k < 8; ++k) amax = fmaxf(amax, fabsf(v[k]));
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) amax = fmaxf(amax, __shfl_xor(amax, d));
    if constexpr (WAVES > 1) {
        if (tid % 64 == 0) part[wave] = amax;
        __syncthreads();  // (and every lane has read the old scale)
#pragma unroll
        for (int w = 0; w < WAVES; ++w) amax = fmaxf(amax, part[w]);
    }
    if (!(old > 0.f && old <= 0x1p100f)) old = 0.f;  // no scale that a write leaves: the earlier slots hold nothing
    const float scale = fmaxf(page_scale(amax), old), inverse = 1.0f / scale;
    if (tid == 0) *scale_at = scale;
    // The earlier tokens' codes move to the new scale, a byte per lane and turn, each load behind the store before it: what a decoding step costs where a page's
    // scale grows (16 sequences x 8 heads, 64 x 128 pages, slots 30 to 60: 33 us, 3 where none grows; slots 100 to 127 of 128 x 256: 128).
    if (slot0 > 0 && scale != old) {
        const float move = old * inverse;
        const int n = slot0 * D;
        for (int i = tid; i < n; i += LANES) {
            uint8_t* at = half ? codes + (i / slot0) * P + i % slot0 : codes + i;
            *at = old == 0.f ? 0 : (uint8_t)to_e4m3x4(e4m3_to_f32(*at) * move, 0.f, 0.f, 0.f);
        }
    }
    // v: a few tokens byte by byte, many turned through LDS
    const bool few = slot1 - slot0 <= 8;
    auto write = [&](int i, v8f_q v) {
        v *= inverse;
        const uint32_t w0 = to_e4m3x4(v[0], v[1], v[2], v[3]), w1 = to_e4m3x4(v[4], v[5], v[6], v[7]);
        const int slot = slot0 + (i >> chunks_log2), ch = i & (chunks - 1);
        if (!half) {
            *reinterpret_cast<v2i*>(codes + slot * D + 8 * ch) = v2i{(int)w0, (int)w1};
        } else if (few) {
#pragma unroll
            for (int k = 0; k < 8; ++k) codes[(8 * ch + k) * P + slot] = (uint8_t)((k < 4 ? w0 : w1) >> (8 * (k & 3)));
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) lds[(8 * ch + k) * v_pad + slot] = (uint8_t)((k < 4 ? w0 : w1) >> (8 * (k & 3)));
        }
    };
    if (tid < count) write(tid, held);
    for (int i = tid + LANES; i < count; i += LANES) write(i, element(i));
    if (half && !few) {
        lds_written<WAVES>();
        const int words_log2 = c.page_log2 - 2;
        for (int i = tid; i < D << words_log2; i += LANES) {
            const int d = i >> words_log2, s = 4 * (i & (P / 4 - 1));
            if (s + 4 <= slot0 || s >= slot1) continue;
            const uint32_t w = *reinterpret_cast<const uint32_t*>(lds + d * v_pad + s);
            if (s >= slot0 && s + 4 <= slot1) {
                *reinterpret_cast<uint32_t*>(codes + d * P + s) = w;
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (s + k >= slot0 && s + k < slot1) codes[d * P + s + k] = (uint8_t)(w >> (8 * k));
            }
        }
    }
}

// Reading: element = code * scale (one fp32 product, rounded once).  A workgroup per 64 tokens of a sequence, head and half, whatever the
// page: 16-token pages one by one would make workgroups that are all latency.  k's rows are widened straight away; v's are turned in
// 4 x 4 blocks of bytes in registers, then through LDS.
// 16 bytes of output: four or eight elements, from one or two dwords of codes.
template <typename T>
__device__ __forceinline__ void store_widened(T* at, v2i codes, float scale) {
    typedef float v2f __attribute__((ext_vector_type(2)));
    typedef T vecT __attribute__((ext_vector_type(16 / sizeof(T))));
    v8f_q y;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const v2f lo = __builtin_amdgcn_cvt_pk_f32_fp8(codes[h], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(codes[h], true);
        y[4 * h] = lo[0] * scale, y[4 * h + 1] = lo[1] * scale, y[4 * h + 2] = hi[0] * scale, y[4 * h + 3] = hi[1] * scale;
    }
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<v4f*>(at) = __builtin_shufflevector(y, y, 0, 1, 2, 3);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {  // the product is rounded on its own, then converted (no single-rounding mixed-precision multiplication)
            float t = y[i];
            asm("" : "+v"(t));
            y[i] = t;
        }
        *reinterpret_cast<vecT*>(at) = __builtin_convertvector(y, vecT);
    }
}

// The place of 16-byte chunk `chunk` of a token's row in LDS: what neighbouring lanes write, four tokens 16 apart, goes to different banks.
__device__ __forceinline__ int turned_chunk(int token, int chunk, int chunks) { return chunk ^ ((2 * (token >> 4)) & (chunks - 1)); }

template <typename T>
__global__ void __launch_bounds__(256) kv_read_kernel(const KvReadParams p) {
    extern __shared__ __align__(16) uint8_t lds[];  // v: 64 tokens' rows of D codes
    const KvCache& c = p.c;
    const int tid = (int)threadIdx.x, P = 1 << c.page_log2, D = c.dim, chunks = D / 16;
    const int half = (int)blockIdx.x & 1, unit = (int)blockIdx.x >> 1, head = unit % c.heads;
    const SeqItem f = find_sequence(c, unit / c.heads, [](int n, int) { return (n + 63) >> 6; });
    if (f.seq < 0) return;
    const int64_t begin = (int64_t)f.item * 64, capacity = (int64_t)c.width << c.page_log2;
    const int n = (int)min(min((int64_t)f.n, capacity) - begin, (int64_t)64);
    if (n <= 0) return;
    const int* row = c.table + (int64_t)f.seq * c.width;
    const uint8_t* codes = half ? c.v : c.k;
    const float* scales = half ? c.v_scale : c.k_scale;
    T* out = (T*)(half ? p.v : p.k) + (((int64_t)f.first + begin) * c.heads + head) * D;
    // the page of a token, or -1 (its row is then left as it was)
    auto page_at = [&](int token) {
        const int page = row[(begin + token) >> c.page_log2];
        return page >= 0 && page < c.pages ? page : -1;
    };
    if (half) {
        for (int i = tid; i < D; i += 256) {  // (a block of four elements, 16 tokens)
            const int four = i >> 2, token = 16 * (i & 3);
            if (token >= n) continue;
            const int page = page_at(token);
            if (page < 0) continue;
            const uint8_t* from = codes + ((int64_t)page * c.heads + head) * ((int64_t)P * D) + 4 * four * P + (int)((begin + token) & (P - 1));
            v4i x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = *reinterpret_cast<const v4i*>(from + e * P);
#pragma unroll
            for (int t4 = 0; t4 < 4; ++t4) {
                const uint32_t a = x[0][t4], b = x[1][t4], d = x[2][t4], e = x[3][t4];  // four tokens of one element each
                const uint32_t ab = __builtin_amdgcn_perm(b, a, 0x05010400), de = __builtin_amdgcn_perm(e, d, 0x05010400),
                               ab2 = __builtin_amdgcn_perm(b, a, 0x07030602), de2 = __builtin_amdgcn_perm(e, d, 0x07030602);
                const uint32_t w[4] = {__builtin_amdgcn_perm(de, ab, 0x05040100), __builtin_amdgcn_perm(de, ab, 0x07060302),
                                       __builtin_amdgcn_perm(de2, ab2, 0x05040100), __builtin_amdgcn_perm(de2, ab2, 0x07060302)};
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const int to = token + 4 * t4 + t;
                    *reinterpret_cast<uint32_t*>(lds + to * D + turned_chunk(to, four >> 2, chunks) * 16 + 4 * (four & 3)) = w[t];
                }
            }
        }
        __syncthreads();
    }
    // 16 bytes of output per lane and store, neighbouring lanes side by side, four loads ahead of their stores.  A wave's lanes are in the same 16
    // tokens (64 E / D of them are 16 at most), so page and scale are scalars.
    constexpr int E = 16 / sizeof(T);
    const int shift = 31 - __clz(D / E), count = n << shift;  // (D / E: a power of two)
    for (int i0 = tid; i0 < count; i0 += 1024) {
        v2i x[4];
        float scale[4];
        int page[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = min(i0 + 256 * u, count - 1), token = i >> shift, e = (i - (token << shift)) * E;
            page[u] = uniform_load(row + ((begin + __builtin_amdgcn_readfirstlane(token)) >> c.page_log2));
            if (page[u] >= c.pages) page[u] = -1;
            const int64_t block = (int64_t)max(page[u], 0) * c.heads + head;
            scale[u] = uniform_load(scales + block);
            auto load = [&](const uint8_t* at) { return E == 8 ? *reinterpret_cast<const v2i*>(at) : v2i{*reinterpret_cast<const int*>(at), 0}; };
            if (half) x[u] = load(lds + token * D + turned_chunk(token, e >> 4, chunks) * 16 + (e & 15));
            else x[u] = load(codes + block * ((int64_t)P * D) + (int)((begin + token) & (P - 1)) * D + e);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = i0 + 256 * u, token = i >> shift;
            if (i < count && page[u] >= 0) store_widened<T>(out + (int64_t)token * c.heads * D + (i - (token << shift)) * E, x[u], scale[u]);
        }
    }
}

}  // namespace

namespace {
struct AppendPlan {
    int64_t items, cache_blocks, blocks, block_waves, q_waves;
    bool single, many;
};
AppendPlan append_plan(const KvAppendParams& p) {
    const KvCache& c = p.c;
    AppendPlan a;
    const int64_t P = (int64_t)1 << c.page_log2;
    a.items = c.rows / P + 2 * (int64_t)c.batch;  // at most: ceil(n / P) + 1 each
    const int64_t units = a.items * c.heads * 2;
    // One wave per page where sequences have up to four new tokens on average, else four, or 16 where that leaves compute units without work
    // and pages and runs are long: a lane's vectors come one after the other.  512 tokens of 8 heads of 128 in pages of 128: 11.8 us with four, 7.7
    // with 16, of 256 20.5 and 11.8; but 2048 of 64 in pages of 64 8.5 and 11.1, runs of 16 tokens 5.0 and 5.9.
    a.single = c.rows <= 4 * (int64_t)c.batch;
    a.many = !a.single && units <= 512 && P * c.dim >= 8192 && (int64_t)c.rows * c.dim >= 4096 * (int64_t)c.batch;
    a.cache_blocks = a.single ? (units + 3) / 4 : units, a.block_waves = a.many ? 16 : 4;
    // q: as many waves for a token as it has 64 vectors, fewer once that makes 8192 in all
    const int64_t vectors = (int64_t)p.q_heads * (c.dim / 8);
    a.q_waves = p.q ? std::max<int64_t>(1, std::min<int64_t>((vectors + 63) / 64, 8192 / c.rows)) : 1;
    a.blocks = a.cache_blocks + (p.q ? (c.rows * a.q_waves + a.block_waves - 1) / a.block_waves : 0);
    return a;
}
int64_t read_blocks(const KvCache& c) { return ((int64_t)c.rows / 64 + c.batch) * c.heads * 2; }

template <typename T>
hipError_t launch_kv_append(const KvAppendParams& p, hipStream_t s) {
    const AppendPlan a = append_plan(p);
    const int v_pad = (1 << p.c.page_log2) + 4;
    const dim3 grid((unsigned)a.blocks), block((unsigned)(64 * a.block_waves));
    const size_t lds = (size_t)p.c.dim * v_pad * (a.single ? 4 : 1);
#define TG_APPEND(WAVES) hipLaunchKernelGGL((kv_append_kernel<T, WAVES>), grid, block, lds, s, p, (int)a.items, (int)a.cache_blocks, v_pad, (int)a.q_waves)
    if (a.single) TG_APPEND(1);
    else if (a.many) TG_APPEND(16);
    else TG_APPEND(4);
#undef TG_APPEND
    return hipGetLastError();
}
}  // namespace

int64_t kv_append_threads(const KvAppendParams& p) {
    const AppendPlan a = append_plan(p);
    return a.blocks * 64 * a.block_waves;
}
int64_t kv_read_threads(const KvReadParams& p) { return read_blocks(p.c) * 256; }

hipError_t run_kv_append(const KvAppendParams& p, bool is_bf16, hipStream_t s) {
    if (p.c.rows <= 0 || p.c.batch <= 0) return hipSuccess;
    return is_bf16 ? launch_kv_append<__bf16>(p, s) : launch_kv_append<_Float16>(p, s);
}

hipError_t run_kv_read(const KvReadParams& p, int out_type, hipStream_t s) {
    const KvCache& c = p.c;
    if (c.rows <= 0 || c.batch <= 0) return hipSuccess;
    const dim3 grid((unsigned)read_blocks(c)), block(256);
    const size_t lds = (size_t)c.dim * 64;
    if (out_type == OUT_BF16) hipLaunchKernelGGL(kv_read_kernel<__bf16>, grid, block, lds, s, p);
    else if (out_type == OUT_F16) hipLaunchKernelGGL(kv_read_kernel<_Float16>, grid, block, lds, s, p);
    else if (out_type == OUT_F32) hipLaunchKernelGGL(kv_read_kernel<float>, grid, block, lds, s, p);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

}  // namespace tg
