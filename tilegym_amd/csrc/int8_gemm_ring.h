// Tiles of 32 x 64 to 256 x 128 of a product in 8-bit integers over a ring of LDS stages, for the row counts between decoding and those that
// fill whole rounds of 256 x 256 tiles, and for the segments of rows that belong to experts: the schedule of fp8_gemm_tile_ring.h over int8 MFMAs.
//
// One workgroup per compute unit: four waves compute (2 x 2), four waves only request the next K steps' slabs by direct global->LDS loads; one
// barrier per step, in front of its last column tiles.  The reasons stand in fp8_gemm_tile_ring.h.  What differs:
//   * the MFMAs are 32x32x32 ones, four to a K step of 128 bytes and output, or in tiles whose steps are loads rather than MFMAs two 16x16x64 ones;
//   * a tile's descriptors start at its own first rows, so that operands may be of any size and a ragged tile's rows anywhere;
//   * K is any multiple of 16: chunks of the last step behind a row's end are requested from beyond the descriptor's range, which makes them
//     zeros in LDS;
//   * partial sums of a split K are int32, and their sum is exact.
#pragma once

#include "int8_device.h"

namespace tg {

#define TG_FENCE() __builtin_amdgcn_sched_barrier(0)

// A computing wave's part of a step: which MFMA, how its fragments lie in LDS, in which order they are multiplied and refilled, and which outputs an
// accumulator register is.  Rows and columns of the part: 16 x 16 or 32 x 32 to an MFMA.

// 16x16x64 MFMAs, two to a step and output: tiles of 32 rows or of up to 64 x 64, whose steps are loads, not MFMAs.
template <int TM, int TN>
struct Mma16 {
    static constexpr int SIDE = 16, VECS = TN / 2;  // vectors of eight columns that a lane has of a row
    static constexpr int WS = 4, LAST = TN == 4 ? 2 : 1;  // weight fragment sets, column tiles behind the barrier
    static_assert(TN == 2 || TN == 4, "column tiles");
    v4i acc[TN][TM];
    v8i af[TM], wf[WS];
    uint32_t frag0, wfrag0;
    int li, lg;
    __device__ __forceinline__ void init(int lane, int row0, int col0, int b_base) {
        li = lane & 15, lg = lane >> 4;
        frag0 = (row0 + li) * kKBlock + ((lg ^ swz16(li)) << 4);
        const int wrow = ((li >> 2) << 3) | (li & 3);
        wfrag0 = b_base + (col0 + wrow) * kKBlock + ((lg ^ swz_w(wrow)) << 4);
#pragma unroll
        for (int tn = 0; tn < TN; ++tn)
#pragma unroll
            for (int tm = 0; tm < TM; ++tm) acc[tn][tm] = v4i{0, 0, 0, 0};
    }
    static __device__ __forceinline__ int a_swizzle(int r) { return swz16(r); }
    static __device__ __forceinline__ int b_swizzle(int r) { return swz_w(r); }
    template <int WGM>
    __device__ __forceinline__ void read_a(int tm, const uint8_t* base) {
        const uint8_t* a = base + tm * (WGM * 16 * kKBlock);
        af[tm] = join(*reinterpret_cast<const v4i*>(a + frag0), *reinterpret_cast<const v4i*>(a + (frag0 ^ 64)));
    }
    __device__ __forceinline__ void read_w(int tn, const uint8_t* base) {
        const uint8_t* b = base + ((tn >> 1) * 32 + (tn & 1) * 4) * kKBlock;
        wf[tn % WS] = join(*reinterpret_cast<const v4i*>(b + wfrag0), *reinterpret_cast<const v4i*>(b + (wfrag0 ^ 64)));
    }
    template <int WGM>
    __device__ __forceinline__ void first(const uint8_t* base) {
        read_w(0, base);
        read_w(1, base);
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) read_a<WGM>(tm, base);
    }
    // column tile by column tile: all row groups' first halves, then the second ones
    __device__ __forceinline__ void before(const uint8_t* cur) {
#pragma unroll
        for (int tn = 0; tn < TN - LAST; ++tn) {
#pragma unroll
            for (int tm = 0; tm < TM; ++tm) {
                acc[tn][tm] = mfma_i8(lo4(wf[tn % WS]), lo4(af[tm]), acc[tn][tm]);
                if (tm == 0 && tn + 2 < TN) read_w(tn + 2, cur);
                TG_FENCE();
            }
#pragma unroll
            for (int tm = 0; tm < TM; ++tm) acc[tn][tm] = mfma_i8(hi4(wf[tn % WS]), hi4(af[tm]), acc[tn][tm]);
            TG_FENCE();
        }
    }
    // row group by row group: the last MFMA of one releases its fragment
    template <int WGM>
    __device__ __forceinline__ void behind(const uint8_t* nxt) {
        read_w(0, nxt);
        if constexpr (TN > 2) read_w(1, nxt);
        TG_FENCE();
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) {
#pragma unroll
            for (int tn = TN - LAST; tn < TN; ++tn) acc[tn][tm] = mfma_i8(lo4(wf[tn % WS]), lo4(af[tm]), acc[tn][tm]);
#pragma unroll
            for (int tn = TN - LAST; tn < TN; ++tn) acc[tn][tm] = mfma_i8(hi4(wf[tn % WS]), hi4(af[tm]), acc[tn][tm]);
            TG_FENCE();
            read_a<WGM>(tm, nxt);
            TG_FENCE();
        }
        if constexpr (TN == 2) read_w(1, nxt);  // (its registers were the last MFMAs')
    }
    __device__ __forceinline__ void keep() {  // (the reads for the step behind the last one)
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) asm volatile("" : : "v"(af[tm]));
        asm volatile("" : : "v"(wf[0]), "v"(wf[1]));
    }
    __device__ __forceinline__ int row() const { return li; }
    __device__ __forceinline__ int column(int v) const { return v * 32 + lg * 8; }
    __device__ __forceinline__ int get(int v, int tm, int i) const { return acc[2 * v + (i >> 2)][tm][i & 3]; }
};

// 32x32x32 MFMAs, four to a step and output.
template <int TM, int TN>
struct Mma32 {
    static constexpr int SIDE = 32, VECS = 2 * TN;
    static_assert(TN == 2 || TN == 3, "column tiles");
    v16i acc[TN][TM];
    v4i af[TM][4], wf[2][4];
    uint32_t frag[4], wfrag[4];
    int li, half;
    __device__ __forceinline__ void init(int lane, int row0, int col0, int b_base) {
        li = lane & 31, half = lane >> 5;
        const int wrow = weight_row_32(li);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            frag[q] = (row0 + li) * kKBlock + (((2 * q + half) ^ swz32(li)) << 4);
            wfrag[q] = b_base + (col0 + wrow) * kKBlock + (((2 * q + half) ^ swz32(wrow)) << 4);
        }
#pragma unroll
        for (int tn = 0; tn < TN; ++tn)
#pragma unroll
            for (int tm = 0; tm < TM; ++tm) acc[tn][tm] = 0;
    }
    static __device__ __forceinline__ int a_swizzle(int r) { return swz32(r); }
    static __device__ __forceinline__ int b_swizzle(int r) { return swz32(r); }
    template <int WGM>
    __device__ __forceinline__ void read_a(int tm, int q, const uint8_t* base) { af[tm][q] = *reinterpret_cast<const v4i*>(base + tm * (WGM * 32 * kKBlock) + frag[q]); }
    __device__ __forceinline__ void read_w(int set, int tn, int q, const uint8_t* base) { wf[set][q] = *reinterpret_cast<const v4i*>(base + tn * (32 * kKBlock) + wfrag[q]); }
    template <int WGM>
    __device__ __forceinline__ void first(const uint8_t* base) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            read_w(0, 0, q, base);
#pragma unroll
            for (int tm = 0; tm < TM; ++tm) read_a<WGM>(tm, q, base);
        }
    }
    __device__ __forceinline__ void before(const uint8_t* cur) {
#pragma unroll
        for (int tn = 0; tn < TN - 1; ++tn)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
#pragma unroll
                for (int tm = 0; tm < TM; ++tm) {
                    acc[tn][tm] = mfma_i8_32(wf[tn & 1][q], af[tm][q], acc[tn][tm]);
                    if (tm == 0) read_w((tn + 1) & 1, tn + 1, q, cur);
                    TG_FENCE();
                }
            }
    }
    // quarter by quarter of the step: its MFMAs release the row groups' pieces, and with three column tiles the weight's
    template <int WGM>
    __device__ __forceinline__ void behind(const uint8_t* nxt) {
        constexpr int set = (TN - 1) & 1;
        if constexpr (set == 1) {
#pragma unroll
            for (int q = 0; q < 4; ++q) read_w(0, 0, q, nxt);
            TG_FENCE();
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
#pragma unroll
            for (int tm = 0; tm < TM; ++tm) acc[TN - 1][tm] = mfma_i8_32(wf[set][q], af[tm][q], acc[TN - 1][tm]);
            TG_FENCE();
            if constexpr (set == 0) read_w(0, 0, q, nxt);
#pragma unroll
            for (int tm = 0; tm < TM; ++tm) read_a<WGM>(tm, q, nxt);
            TG_FENCE();
        }
    }
    __device__ __forceinline__ void keep() {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
#pragma unroll
            for (int tm = 0; tm < TM; ++tm) asm volatile("" : : "v"(af[tm][q]));
            asm volatile("" : : "v"(wf[0][q]));
        }
    }
    __device__ __forceinline__ int row() const { return li; }
    __device__ __forceinline__ int column(int v) const { return v * 16 + half * 8; }
    __device__ __forceinline__ int get(int v, int tm, int i) const { return acc[v >> 1][tm][8 * (v & 1) + i]; }
};

template <int BM, int BN, int STAGES, bool SPLIT, bool RAGGED>
__global__ void __launch_bounds__(512, 1) int8_gemm_ring_kernel(const Int8GemmParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr bool WIDE = BM >= 64 && BN >= 128;
    constexpr int NL = 4, WGN = BN == 32 ? 1 : 2, WGM = 4 / WGN, SIDE = WIDE ? 32 : 16;
    constexpr int WTN = BN / WGN;
    constexpr int TM = BM / (SIDE * WGM), TN = WTN / SIDE;
    using Mma = std::conditional_t<WIDE, Mma32<TM, WIDE ? TN : 2>, Mma16<TM, WIDE ? 2 : TN>>;
    constexpr int VECS = Mma::VECS;
    constexpr int A_IT = BM / (8 * NL), B_IT = BN / (8 * NL);
    constexpr int STAGE_BYTES = (BM + BN) * kKBlock;
    constexpr int PER_STEP = A_IT + B_IT;
    static_assert(BM % (SIDE * WGM) == 0 && STAGES >= 3 && STAGES * STAGE_BYTES <= 160 * 1024, "shape");
    static_assert(!(SPLIT && RAGGED), "K is split for dense rows only");

    __shared__ __align__(1024) uint8_t lds[STAGES * STAGE_BYTES];  // stage s: A slab, then B slab

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int K = p.K;
    const int tiles_n = (p.N + BN - 1) / BN;
    int n0, rows_valid, expert = 0;
    int64_t m0;
    if constexpr (RAGGED) {
        int tile_n;
        if (!ragged_tile<BM, true>(p, (int)blockIdx.x, tiles_n, lane, expert, m0, rows_valid, tile_n)) return;
        n0 = tile_n * BN;
    } else {
        const int tiles_m = (p.M + BM - 1) / BM;
        const int pid = xcd_remap((int)blockIdx.x, tiles_m * tiles_n);
        constexpr int GM = 8;
        const int width = GM * tiles_n;
        const int group = pid / width, first_m = group * GM;
        const int gsz = min(tiles_m - first_m, GM);
        m0 = (int64_t)(first_m + (pid % width) % gsz) * BM;
        n0 = ((pid % width) / gsz) * BN;
        rows_valid = (int)min((int64_t)BM, p.M - m0);
    }
    int ks = 0, ks_end = (K + kKBlock - 1) / kKBlock;
    if constexpr (SPLIT) {
        ks = blockIdx.y * p.ksteps_per_split;
        ks_end = min(ks + p.ksteps_per_split, ks_end);
    }
    const int nsteps = ks_end - ks, last = ks_end - 1;
    if (nsteps <= 0) return;

    constexpr int kPro = (STAGES - 1) * PER_STEP, kLoop = (STAGES - 2) * PER_STEP;  // loads that may stay in flight
    static_assert(kPro < 64, "vmcnt has six bits");
    constexpr int kWaitPro = 0x0F70 | (kPro & 15) | ((kPro >> 4) << 14);
    constexpr int kWaitLoop = 0x0F70 | (kLoop & 15) | ((kLoop >> 4) << 14);
    constexpr int kWaitAll = 0x0F70;
    constexpr int kWaitLds = 0xC07F;

    if (wave >= 4) {
        // ------------------------------------------------------------ loading waves
        const int lw = wave - 4;
        const int lrow = lane >> 3;
        const int lj = (lane & 7) ^ Mma::a_swizzle(((lw & 1) << 3) | lrow);
        const int ljb = (lane & 7) ^ Mma::b_swizzle(((lw & 1) << 3) | lrow);
        constexpr uint32_t kOutOfRange = 0x80000000u;  // beyond the descriptor's 2^31 - 1 bytes
        uint32_t a_off[A_IT], b_off[B_IT];
#pragma unroll
        for (int i = 0; i < A_IT; ++i) a_off[i] = (uint32_t)min((i * NL + lw) * 8 + lrow, rows_valid - 1) * (uint32_t)K + lj * 16;
#pragma unroll
        for (int i = 0; i < B_IT; ++i) b_off[i] = (uint32_t)min((i * NL + lw) * 8 + lrow, p.N - 1 - n0) * (uint32_t)K + ljb * 16;
        const v4i rsrc_a = make_rsrc(p.A + m0 * K), rsrc_b = make_rsrc(p.B + ((int64_t)expert * p.N + n0) * K);
        const uint32_t lds0 = lds_address(lds) + lw * 1024;
        auto issue = [&](int kstep, int stage) {
            const int k0 = min(kstep, last) * kKBlock;
            const uint32_t dst = lds0 + stage * STAGE_BYTES;
            if (k0 + kKBlock <= K) {
#pragma unroll
                for (int i = 0; i < B_IT; ++i) direct_load_b128(rsrc_b, dst + BM * kKBlock + i * NL * 1024, b_off[i], k0);
#pragma unroll
                for (int i = 0; i < A_IT; ++i) direct_load_b128(rsrc_a, dst + i * NL * 1024, a_off[i], k0);
            } else {  // the last step of a K that is no multiple of 128: as many loads
                const bool a_in = k0 + lj * 16 < K, b_in = k0 + ljb * 16 < K;
#pragma unroll
                for (int i = 0; i < B_IT; ++i) direct_load_b128(rsrc_b, dst + BM * kKBlock + i * NL * 1024, b_in ? b_off[i] : kOutOfRange, k0);
#pragma unroll
                for (int i = 0; i < A_IT; ++i) direct_load_b128(rsrc_a, dst + i * NL * 1024, a_in ? a_off[i] : kOutOfRange, k0);
            }
        };
#pragma unroll
        for (int s = 0; s < STAGES; ++s) issue(ks + s, s);
        __builtin_amdgcn_s_waitcnt(kWaitPro);
        __builtin_amdgcn_s_barrier();
        int stage = 0;
        for (int k = 0; k < nsteps; ++k) {
            __builtin_amdgcn_s_waitcnt(kWaitLoop);  // step k+1 has landed (steps past the end re-fetch the last one)
            __builtin_amdgcn_s_barrier();           // and every computing wave has read step k
            issue(ks + k + STAGES, stage);
            stage = stage == STAGES - 1 ? 0 : stage + 1;
        }
        __builtin_amdgcn_s_waitcnt(kWaitAll);  // the re-fetches past the end must land before the workgroup's LDS is released
        return;
    }

    // ---------------------------------------------------------------- computing waves
    const int wm = wave % WGM, wn = wave / WGM;
    Mma mma;
    mma.init(lane, wm * SIDE, wn * WTN, BM * kKBlock);
    const int li = mma.row();

    // the scales of this lane's rows, asked for in front of the K loop
    const float* sb = p.sb + (int64_t)expert * p.N * p.sb_step;
    float srow[TM];
#pragma unroll
    for (int tm = 0; tm < TM; ++tm) srow[tm] = p.sa[(m0 + min((tm * WGM + wm) * SIDE + li, rows_valid - 1)) * p.sa_step];

    __builtin_amdgcn_s_barrier();  // step 0 has landed
    mma.template first<WGM>(lds);
    int stage = 0;
    for (int k = 0; k < nsteps; ++k) {
        const uint8_t* cur = lds + stage * STAGE_BYTES;
        stage = stage == STAGES - 1 ? 0 : stage + 1;
        const uint8_t* nxt = lds + stage * STAGE_BYTES;
        TG_FENCE();
        mma.before(cur);
        __builtin_amdgcn_s_waitcnt(kWaitLds);  // all my reads of step k are done
        __builtin_amdgcn_s_barrier();          // step k+1 is visible
        TG_FENCE();
        mma.template behind<WGM>(nxt);
    }
    mma.keep();

    const int col0 = n0 + wn * WTN;
    if constexpr (SPLIT) {
        int* mine = p.partials + (int64_t)blockIdx.y * p.M * p.N;
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) {
            const int rt = (tm * WGM + wm) * SIDE + li;
            if (rt >= rows_valid) continue;
#pragma unroll
            for (int v = 0; v < VECS; ++v) {
                const int col = col0 + mma.column(v);
                int* to = mine + (m0 + rt) * p.N + col;
                if (p.N % 8 == 0) {
                    if (col >= p.N) continue;
                    *reinterpret_cast<v4i*>(to) = v4i{mma.get(v, tm, 0), mma.get(v, tm, 1), mma.get(v, tm, 2), mma.get(v, tm, 3)};
                    *reinterpret_cast<v4i*>(to + 4) = v4i{mma.get(v, tm, 4), mma.get(v, tm, 5), mma.get(v, tm, 6), mma.get(v, tm, 7)};
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (col + i < p.N) to[i] = mma.get(v, tm, i);
                }
            }
        }
        return;
    }
    auto emit_whole = [&](auto type_tag) __attribute__((always_inline)) {
        constexpr int OT = decltype(type_tag)::value;
        constexpr int FT = TM * VECS > 16 ? 2 : VECS;  // vectors whose factors are in registers at a time
#pragma unroll
        for (int v0 = 0; v0 < VECS; v0 += FT) {
            AnyColumnFactors f[FT];
#pragma unroll
            for (int v = 0; v < FT; ++v) f[v].load(p, sb, min(col0 + mma.column(v0 + v), p.N - 8));
#pragma unroll
            for (int tm = 0; tm < TM; ++tm) {
                const int rt = (tm * WGM + wm) * SIDE + li;
                if (rt >= rows_valid) continue;
#pragma unroll
                for (int v = 0; v < FT; ++v) {
                    const int col = col0 + mma.column(v0 + v);
                    if (col >= p.N) continue;
                    v4f x, y;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        x[r] = f[v].finished(mma.get(v0 + v, tm, r), srow[tm], r);
                        y[r] = f[v].finished(mma.get(v0 + v, tm, 4 + r), srow[tm], 4 + r);
                    }
                    put8<OT>(p.C, (m0 + rt) * p.ldc + col, x, y);
                }
            }
        }
    };
    if (p.vec_store) {
        if (p.out_type == OUT_BF16) emit_whole(std::integral_constant<int, OUT_BF16>{});
        else if (p.out_type == OUT_F32) emit_whole(std::integral_constant<int, OUT_F32>{});
        else emit_whole(std::integral_constant<int, OUT_F16>{});
        return;
    }
    // rows of outputs that are no whole vectors: element by element
#pragma unroll
    for (int v = 0; v < VECS; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int col = col0 + mma.column(v) + i;
            if (col >= p.N) continue;
            const float s = sb[(int64_t)col * p.sb_step], b = load_bias(p.bias, p.bias_type, col);
#pragma unroll
            for (int tm = 0; tm < TM; ++tm) {
                const int rt = (tm * WGM + wm) * SIDE + li;
                if (rt < rows_valid) put1(p, (m0 + rt) * p.ldc + col, finish(mma.get(v, tm, i), srow[tm], s, b));
            }
        }
#endif
}

template <int BM, int BN, int STAGES>
inline hipError_t launch_int8_ring(const Int8GemmParams& p, hipStream_t stream) {
    const int64_t cols = ((int64_t)p.N + BN - 1) / BN;
    // ragged: no more row tiles than M rows in E segments can have
    const int64_t tiles = cols * (p.m_indptr ? (int64_t)p.M / BM + (p.E < p.M ? p.E : p.M) : ((int64_t)p.M + BM - 1) / BM);
    if (tiles * p.split_k * 512 > kMostThreads) return hipErrorInvalidValue;
    const dim3 grid((unsigned)tiles, p.split_k), block(512);
    if (p.m_indptr) hipLaunchKernelGGL((int8_gemm_ring_kernel<BM, BN, STAGES, false, true>), grid, block, 0, stream, p);
    else if (p.split_k > 1) hipLaunchKernelGGL((int8_gemm_ring_kernel<BM, BN, STAGES, true, false>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((int8_gemm_ring_kernel<BM, BN, STAGES, false, false>), grid, block, 0, stream, p);
    return hipGetLastError();
}

#undef TG_FENCE

}  // namespace tg
