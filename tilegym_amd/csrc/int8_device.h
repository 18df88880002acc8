// Device-side building blocks of the products in 8-bit integers: C[m,n] = sa[m] * sb[n] * sum_k A[m,k] * B[n,k] + bias[n].
//
// The sums are 32-bit integers, so they are exact (|a b| <= 2^14, K <= 131071) and the same whatever the tile, the split and the order; every
// kernel ends in the same fp32 steps (finish), so all of them return the same bits.
#pragma once
#include "fp8_gemm_tile.h"
#include "tg_host.h"

namespace tg {

// Two 16x16x64 int8 MFMAs over the 128 bytes of K that an e4m3 16x16x128 MFMA takes, with the same operand layout: lane l holds
// 16-byte chunks l / 16 and l / 16 + 4 of row l % 16.
__device__ __forceinline__ v4i mfma_i8(v4i w, v4i x, v4i acc) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(w, x, acc, 0, 0, 0); }

// A 32x32x32 int8 MFMA: lane l holds 16 bytes of row l % 32, those of K half l / 32; a lane gets column l % 32 and, in register 4 g + j, row
// 8 g + 4 (l / 32) + j.  It issues at the matrix pipe's full rate, where two waves on a SIMD get 0.71 and one gets 0.58 of it out of 16x16x64 ones
// (registers only, zeros: 4966, 3531, 2900 TOP/s; normally distributed codes, at the power limit: 3507, 3175, 2879).
typedef int v16i __attribute__((ext_vector_type(16)));
__device__ __forceinline__ v16i mfma_i8_32(v4i w, v4i x, v16i acc) { return __builtin_amdgcn_mfma_i32_32x32x32_i8(w, x, acc, 0, 0, 0); }
// The weight row (of 32) that is row r of such an MFMA: bits 2 and 3 change places, so that registers 0 ... 7 and 8 ... 15 of a lane are eight
// consecutive columns of the output each, 8 (l / 32) and 16 + 8 (l / 32) on.
__device__ __forceinline__ int weight_row_32(int r) { return (r & 19) | ((r & 4) << 1) | ((r & 8) >> 1); }

// Chunk swizzle of a slab whose fragments are read 32 rows at a time: 16-byte chunk j of row r sits at position j ^ swz32(r).  A 16-byte read serves lanes
// 0 - 3, 12 - 15 and 20 - 27 of each half wave together, then the others: the rows of one parity among them, which share 32 of the 64 banks, differ in
// bits 1 to 3.
__device__ __forceinline__ int swz32(int r) { return (r >> 1) & 7; }

// One output from its integer sum.  Three roundings at most beside the store's: the sum's conversion (exact to 2^24), the product with the
// token's scale, and one multiply-add with the channel's scale and the bias.  Where there is none, kNoBias makes it the product alone: a product of -0 stays
// one, which + 0 would not leave it.
__device__ __forceinline__ float finish(int sum, float sa, float sb, float bias) { return __builtin_fmaf((float)sum * sa, sb, bias); }
[[maybe_unused]] constexpr float kNoBias = -0.f;

template <typename T>
__device__ __forceinline__ float load_any(const void* p, int64_t i) { return (float)((const T*)p)[i]; }
__device__ __forceinline__ float load_bias(const void* p, int type, int64_t i) {
    if (!p) return kNoBias;
    return type == OUT_F32 ? load_any<float>(p, i) : type == OUT_BF16 ? load_any<__bf16>(p, i) : load_any<_Float16>(p, i);
}

// Rows of expert e.  Rows outside the M that a and c have are nobody's, whatever m_indptr holds.
__device__ __forceinline__ int ragged_rows(const Int8GemmParams& p, int e) {
    const int lo = p.m_indptr[e], hi = min(p.m_indptr[e + 1], p.M);
    return lo >= 0 && hi > lo ? hi - lo : 0;
}

// Workgroup `bid`'s tile of the experts' BM-row tiles x tiles_n columns of them; false: none is left for it.  An expert's row tiles come one after the
// other over the same columns, which they read the same weight rows for.  Every lane of a wave gets the same.
template <int BM>
__device__ __forceinline__ bool ragged_tile(const Int8GemmParams& p, int bid, int tiles_n, int lane, int& expert, int64_t& m0, int& rows_valid, int& tile_n) {
    auto scan = [&](int e0, int& rows) {  // row tiles of the experts from e0 up to and with the lane's
        rows = e0 + lane < p.E ? ragged_rows(p, e0 + lane) : 0;
        int upto = (rows + BM - 1) / BM;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int t = __shfl_up(upto, d);
            if (lane >= d) upto += t;
        }
        return upto;
    };
    int rows = 0, upto = scan(0, rows), total = __shfl(upto, 63);
    for (int e0 = 64; e0 < p.E; e0 += 64) {
        int more;
        total += __shfl(scan(e0, more), 63);
    }
    total = __builtin_amdgcn_readfirstlane(total) * tiles_n;
    if (bid >= total) return false;
    const int row_tile = bid / tiles_n;
    int base = 0, e0 = 0;
    unsigned long long hit;
    while (!(hit = __ballot(base + upto > row_tile))) {
        base += __shfl(upto, 63);
        e0 += 64;
        upto = scan(e0, rows);
    }
    const int l = __ffsll((long long)hit) - 1;
    expert = __builtin_amdgcn_readfirstlane(e0 + l);
    rows = __builtin_amdgcn_readlane(rows, l);
    const int mine = (rows + BM - 1) / BM, first = __builtin_amdgcn_readfirstlane(base) + __builtin_amdgcn_readlane(upto, l) - mine;
    const int inside = bid - first * tiles_n;  // of this expert's mine * tiles_n tiles
    const int at = (inside % mine) * BM;
    tile_n = inside / mine;
    m0 = (int64_t)p.m_indptr[expert] + at;
    rows_valid = min(BM, rows - at);
    return true;
}

// The same for a workgroup that takes one tile after the other, in their order: 64 experts' row tiles stay in registers, so that finding the next
// tile reads memory only where it belongs to a later 64.
template <int BM>
struct RaggedWalk {
    int upto, rows, first;  // lane l: the row tiles of experts e0 ... e0 + l, expert e0 + l's rows and the first of them
    int e0, base;           // base: row tiles of the experts in front of e0
    __device__ __forceinline__ void scan(const Int8GemmParams& p, int lane) {
        const int e = e0 + lane;
        rows = e < p.E ? ragged_rows(p, e) : 0;
        first = e < p.E ? p.m_indptr[e] : 0;
        upto = (rows + BM - 1) / BM;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int t = __shfl_up(upto, d);
            if (lane >= d) upto += t;
        }
    }
    // All tiles there are, as far as the host counted them: segments that overlap would have more, and their sum need not stay within 32 bits.
    __device__ __forceinline__ int start(const Int8GemmParams& p, int lane, int tiles_n) {
        const int most = (int)most_row_tiles(p.M, p.E, BM);
        int total = 0;
        for (e0 = (p.E - 1) / 64 * 64;; e0 -= 64) {
            scan(p, lane);
            total = min(total + __builtin_amdgcn_readlane(upto, 63), most);
            if (e0 == 0) break;
        }
        base = 0;
        return total * tiles_n;
    }
    // Tile pid, below that total and not below the last one asked for (see walking_grid).
    __device__ __forceinline__ void find(const Int8GemmParams& p, int lane, int pid, int tiles_n, int& expert, int& m0, int& rows_valid, int& tile_n) {
        const int row_tile = pid / tiles_n;
        unsigned long long hit;
        while (!(hit = __ballot(base + upto > row_tile))) {
            base += __builtin_amdgcn_readlane(upto, 63);
            e0 += 64;
            scan(p, lane);
        }
        const int l = __builtin_amdgcn_readfirstlane(__ffsll((long long)hit) - 1), has = __builtin_amdgcn_readlane(rows, l);
        const int mine = (has + BM - 1) / BM, inside = pid - (base + __builtin_amdgcn_readlane(upto, l) - mine) * tiles_n;
        const int at = inside % mine * BM;
        expert = e0 + l;
        tile_n = inside / mine;
        m0 = __builtin_amdgcn_readlane(first, l) + at;
        rows_valid = min(BM, has - at);
    }
};

// Stores of eight outputs at byte offsets from a tile's first row; those from kBeyond on are left out.
constexpr uint32_t kBeyond = 0x80000000u;
struct StoreTile {
#if defined(__HIP_DEVICE_COMPILE__)
    __amdgpu_buffer_rsrc_t rsrc;
    __device__ __forceinline__ StoreTile(void* base, int64_t offset) : rsrc(__builtin_amdgcn_make_buffer_rsrc((char*)base + offset, 0, 0x7FFFFFFF, 0x00020000)) {}
    template <int OT>
    __device__ __forceinline__ void put8(uint32_t at, v4f lo, v4f hi) const {
        typedef float v8f __attribute__((ext_vector_type(8)));
        typedef uint32_t v4u __attribute__((ext_vector_type(4)));
        const v8f v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        if constexpr (OT == OUT_F32) {
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u, lo), rsrc, at, 0, 0);
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u, hi), rsrc, at | 16, 0, 0);
        } else if constexpr (OT == OUT_BF16) {
            typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u, __builtin_convertvector(v, bf16x8)), rsrc, at, 0, 0);
        } else {
            typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u, __builtin_convertvector(v, f16x8)), rsrc, at, 0, 0);
        }
    }
#endif
};

// One output at element `to` of C.
__device__ __forceinline__ void put1(const Int8GemmParams& p, int64_t to, float y) {
    if (p.out_type == OUT_BF16) ((__bf16*)p.C)[to] = (__bf16)y;
    else if (p.out_type == OUT_F16) ((_Float16*)p.C)[to] = (_Float16)y;
    else ((float*)p.C)[to] = y;
}

__device__ __forceinline__ v4i lo4(v8i v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3); }
__device__ __forceinline__ v4i hi4(v8i v) { return __builtin_shufflevector(v, v, 4, 5, 6, 7); }

// Scales and biases of the eight columns from `col` on, a multiple of eight (vec_store).
enum BiasKind { BIAS_NONE = 0, BIAS_F32 = 1, BIAS_16 = 2 };
inline int bias_kind(const Int8GemmParams& p) { return !p.bias ? BIAS_NONE : p.bias_type == OUT_F32 ? BIAS_F32 : BIAS_16; }
template <int BIAS>
struct ColumnFactors {
#if defined(__HIP_DEVICE_COMPILE__)
    float s[8], b[BIAS ? 8 : 1];
    // the output in column i of them from its integer sum
    __device__ __forceinline__ float finished(int sum, float sa, int i) const { return finish(sum, sa, s[i], BIAS ? b[BIAS ? i : 0] : kNoBias); }
    __device__ __forceinline__ void load_scales(const Int8GemmParams& p, const float* sb, int col) {
        if (p.sb_step) {
            const v4f x = *reinterpret_cast<const v4f*>(sb + col), y = *reinterpret_cast<const v4f*>(sb + col + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] = x[i], s[4 + i] = y[i];
        } else {
            const float x = *sb;
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] = x;
        }
    }
    // (no branches: StoreTile's reason)
    __device__ __forceinline__ void load_bias8(const Int8GemmParams& p, int col) {
        if constexpr (BIAS == BIAS_F32) {
            const v4f u = *reinterpret_cast<const v4f*>((const float*)p.bias + col), v = *reinterpret_cast<const v4f*>((const float*)p.bias + col + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) b[i] = u[i], b[4 + i] = v[i];
        } else if constexpr (BIAS == BIAS_16) {
            typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
            typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
            const u16x8 u = *reinterpret_cast<const u16x8*>((const uint16_t*)p.bias + col);
            const f16x8 h = __builtin_bit_cast(f16x8, u);
#pragma unroll
            for (int i = 0; i < 8; ++i) b[i] = p.bias_type == OUT_BF16 ? __uint_as_float((uint32_t)u[i] << 16) : (float)h[i];
        }
    }
#endif
};

}  // namespace tg
