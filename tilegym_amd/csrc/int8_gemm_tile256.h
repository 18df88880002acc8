// 256 x 256 tiles of a product in 8-bit integers, persistent, with a hand-ordered K loop (prompts): the schedule of fp8_gemm_tile256.h over
// int8 MFMAs.
//
// Four waves, one per SIMD, each with a 128 x 128 part of the tile, one workgroup per compute unit that walks tiles b, b + grid, ... of the rastered
// sequence; two activation slabs and three weight slabs (160 KiB, all of LDS); requests two steps ahead, running on into the next tile; one barrier per
// step in front of its last sixteen MFMAs.  The reasons stand in fp8_gemm_tile256.h.  What differs: 32x32x32 MFMAs, four to a K step and output tile, and an
// epilogue with a scale per row and per column and a bias.
// Bound by power: 8192 x 28672 x 4096 takes 760 to 810 us (2.4 to 2.5 POP/s) with the MFMAs busy 71 % of the cycles; short K by the outputs, 7.6 us for each round of tiles.
//
// Over experts the same kernel walks the experts' row tiles (RaggedWalk); 24576 rows over 64 experts of (2816, 2048): 176 to 189 us, of (2048, 1408): 98 to 108, a third of
// it for rows that the last tile of an expert does not have.
// K must be a multiple of 128 and at least 256, the operands below 2 GiB each, the outputs in whole vectors (vec_store).
#pragma once

#include "int8_device.h"

namespace tg {

// One element of an accumulator, out of the accumulation register it is in: left to itself the compiler copies whole accumulators out of them at the end
// of the K loop, more than the other registers hold.  The caller sees to the wait states behind the MFMA that wrote it.
__device__ __forceinline__ int read_acc(int x) {
    int y;
    asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(y) : "a"(x));
    return y;
}

// A kernel per output type and kind of bias: with all in one the compiler reads every
// accumulator out in front of the choice, spills, and waits for the reload in every K step (855 -> 1006 us).
template <int OT, int BIAS, bool RAGGED>
__global__ void __launch_bounds__(256, 1) int8_gemm_tile256_kernel(const Int8GemmParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int BM = 256, BN = 256, WGM = 2, WGN = 2, NW = 4;
    constexpr int WTN = BN / WGN;
    constexpr int TM = 4, TN = WTN / 32;          // 4 row groups x 4 column tiles of 32 x 32 per wave
    constexpr int SLAB = 256 * kKBlock;
    constexpr int A_STAGES = 2, B_STAGES = 3;
    constexpr int IT = 256 / (8 * NW);
    static_assert(TN == 4 && IT == 8, "schedule below is written for 4 x 4 MFMA tiles and 8 + 8 loads per wave");

    __shared__ __align__(1024) uint8_t sA[A_STAGES * SLAB];
    __shared__ __align__(1024) uint8_t sB[B_STAGES * SLAB];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave % WGM, wn = wave / WGM;
    const int K = p.K;
    const int tiles_n = (p.N + BN - 1) / BN, tiles_m = (p.M + BM - 1) / BM, stride = (int)gridDim.x;
    RaggedWalk<BM> walk;
    int total;
    if constexpr (RAGGED) total = walk.start(p, lane, tiles_n);
    else total = tiles_m * tiles_n;
    int rows = BM, expert = 0;  // of the tile at (m0, n0)
    auto origin = [&](int v, int& om0, int& on0) {
        const int pid = xcd_remap(v, total);
        if constexpr (RAGGED) {
            int tile_n;
            walk.find(p, lane, pid, tiles_n, expert, om0, rows, tile_n);
            on0 = tile_n * BN;
            return;
        }
        constexpr int GM = 8;
        const int width = GM * tiles_n;
        const int group = pid / width, first_m = group * GM;
        const int gsz = min(tiles_m - first_m, GM);
        om0 = (first_m + (pid % width) % gsz) * BM;
        on0 = ((pid % width) / gsz) * BN;
        rows = min(BM, p.M - om0);
    };
    int vt = (int)blockIdx.x;
    if (RAGGED && vt >= total) return;
    int m0, n0;
    origin(vt, m0, n0);
    const int nsteps = K / kKBlock, last = nsteps - 1;

    const int lrow = lane >> 3;
    const int lj = (lane & 7) ^ swz32(((wave & 1) << 3) | lrow);
    uint32_t a_off[IT], b_off[IT];
    auto set_offsets = [&](int om0, int on0) {
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int r = (i * NW + wave) * 8 + lrow;
            a_off[i] = (uint32_t)(om0 + min(r, rows - 1)) * (uint32_t)K + lj * 16;
            b_off[i] = (uint32_t)min(on0 + r, p.N - 1) * (uint32_t)K + lj * 16;
        }
    };
    set_offsets(m0, n0);
    const v4i rsrc_a = make_rsrc(p.A);
    v4i rsrc_b = make_rsrc(p.B + (int64_t)expert * p.N * K);
    const uint32_t ldsA = settle(lds_address(sA) + wave * 1024), ldsB = settle(lds_address(sB) + wave * 1024);
    auto load_a = [&](int i, int kstep, int stage) {
        direct_load_b128_settled(rsrc_a, ldsA + stage * SLAB + i * NW * 1024, a_off[i], kstep * kKBlock);
    };
    auto load_b = [&](int i, int kstep, int stage) {
        direct_load_b128_settled(rsrc_b, ldsB + stage * SLAB + i * NW * 1024, b_off[i], kstep * kKBlock);
    };

    // chunk 2 q + half of a row is the lane's share of the K step's q-th 32 bytes
    const int li = lane & 31, half = lane >> 5;
    const int wrow = weight_row_32(li);
    uint32_t frag[4], wfrag[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        frag[q] = (wm * 32 + li) * kKBlock + (((2 * q + half) ^ swz32(li)) << 4);
        wfrag[q] = (wn * WTN + wrow) * kKBlock + (((2 * q + half) ^ swz32(wrow)) << 4);
    }
    auto read_a = [&](int tm, int q, const uint8_t* cA) { return *reinterpret_cast<const v4i*>(cA + tm * (WGM * 32 * kKBlock) + frag[q]); };
    auto read_w = [&](int tn, int q, const uint8_t* cB) { return *reinterpret_cast<const v4i*>(cB + tn * (32 * kKBlock) + wfrag[q]); };

    v16i acc[TN][TM];
#pragma unroll
    for (int tn = 0; tn < TN; ++tn)
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) acc[tn][tm] = 0;

    constexpr int kWaitBut16 = 0x4F70 | 0, kWaitBut8 = 0x0F70 | 8, kWaitAll = 0x0F70;
    constexpr int kWaitLds = 0xC07F;
#define TG_FENCE() __builtin_amdgcn_sched_barrier(0)

#pragma unroll
    for (int i = 0; i < IT; ++i) load_a(i, 0, 0);
#pragma unroll
    for (int i = 0; i < IT; ++i) load_b(i, 0, 0);
#pragma unroll
    for (int i = 0; i < IT; ++i) load_b(i, min(1, last), 1);
#pragma unroll
    for (int i = 0; i < IT; ++i) load_a(i, min(1, last), 1);
    __builtin_amdgcn_s_waitcnt(kWaitBut16);
    __builtin_amdgcn_s_barrier();
    v4i af[TM][4], wf[2][4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        wf[0][q] = read_w(0, q, sB);
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) af[tm][q] = read_a(tm, q, sA);
    }

    int sa = 0, sb = 0;
    for (;;) {
        const int cm0 = m0, cn0 = n0, rows_valid = rows;
        const float* const sb_tile = p.sb + (int64_t)expert * p.N * p.sb_step;
        bool more = false;
        // the tile's scales, asked for here: a trip to memory in front of the stores would be time without MFMAs
        float srow[TM];
        ColumnFactors<BIAS> scale[2 * TN];
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) srow[tm] = p.sa[(int64_t)(cm0 + min((tm * WGM + wm) * 32 + li, rows_valid - 1)) * p.sa_step];
#pragma unroll
        for (int t = 0; t < 2 * TN; ++t) scale[t].load_scales(p, sb_tile, min(cn0 + wn * WTN + t * 16 + half * 8, p.N - 8));
        for (int k = 0; k < nsteps; ++k) {
            if (k == nsteps - 2) {
                more = vt + stride < total;
                if (more) {
                    vt += stride;
                    origin(vt, m0, n0);
                    set_offsets(m0, n0);
                    if constexpr (RAGGED) rsrc_b = make_rsrc(p.B + (int64_t)expert * p.N * K);
                }
            }
            int k2 = k + 2;
            if (k2 >= nsteps) k2 = more ? k2 - nsteps : last;
            const int sa1 = sa ^ 1;
            const int sb1 = sb == B_STAGES - 1 ? 0 : sb + 1;
            const int sb2 = sb1 == B_STAGES - 1 ? 0 : sb1 + 1;
            const uint8_t* cB = sB + sb * SLAB;
            TG_FENCE();
            // column tiles 0 .. 2 in groups of four MFMAs, one per row group; behind each of the first eight groups a direct load, behind a tile's
            // first two the next one's weight fragment, so that the barrier finds no read under way
#pragma unroll
            for (int tn = 0; tn < TN - 1; ++tn) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
#pragma unroll
                    for (int tm = 0; tm < TM; ++tm) acc[tn][tm] = mfma_i8_32(wf[tn & 1][q], af[tm][q], acc[tn][tm]);
                    TG_FENCE();
                    if (4 * tn + q < IT) load_b(4 * tn + q, k2, sb2);
                    if (q < 2) {
                        wf[(tn + 1) & 1][2 * q] = read_w(tn + 1, 2 * q, cB);
                        wf[(tn + 1) & 1][2 * q + 1] = read_w(tn + 1, 2 * q + 1, cB);
                    }
                    TG_FENCE();
                }
            }
            __builtin_amdgcn_s_waitcnt(kWaitBut8);
            __builtin_amdgcn_s_waitcnt(kWaitLds);
            __builtin_amdgcn_s_barrier();
            TG_FENCE();
            // column tile 3: each MFMA releases a piece of an activation fragment, which is refilled from A(k+1) at once
            const uint8_t* nA = sA + sa1 * SLAB;
            const uint8_t* nB = sB + sb1 * SLAB;
#pragma unroll
            for (int q = 0; q < 4; ++q) wf[0][q] = read_w(0, q, nB);
            TG_FENCE();
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    acc[TN - 1][2 * t] = mfma_i8_32(wf[1][q], af[2 * t][q], acc[TN - 1][2 * t]);
                    acc[TN - 1][2 * t + 1] = mfma_i8_32(wf[1][q], af[2 * t + 1][q], acc[TN - 1][2 * t + 1]);
                    TG_FENCE();
                    af[2 * t][q] = read_a(2 * t, q, nA);
                    af[2 * t + 1][q] = read_a(2 * t + 1, q, nA);
                    load_a(2 * q + t, k2, sa);
                    TG_FENCE();
                }
            sa = sa1;
            sb = sb1;
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
#pragma unroll
            for (int tm = 0; tm < TM; ++tm) asm volatile("" : : "v"(af[tm][q]));
            asm volatile("" : : "v"(wf[0][q]));
        }

        // ---- epilogue, straight from the accumulators
        // (stores without branches, those outside the matrix beyond the descriptor's range: around a branch the compiler copies whole accumulators out
        // of the accumulation registers early, more than the others hold)
        constexpr int SIZE = OT == OUT_F32 ? 4 : 2;
        const StoreTile out(p.C, (int64_t)cm0 * p.ldc * SIZE);
        uint32_t dsts[TM];
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) {
            const int rt = (tm * WGM + wm) * 32 + li;
            dsts[tm] = rt < rows_valid ? (uint32_t)rt * (uint32_t)(p.ldc * SIZE) : kBeyond;
        }
        asm volatile("s_nop 15\n\ts_nop 15");  // (the last MFMAs' results, in front of read_acc: 18 wait states)
        TG_FENCE();
        // row group by row group: the sixteens of columns that make a line follow one another.  Biases: a line's sixteens at a time
        auto group = [&](auto group_tag) __attribute__((always_inline)) {
            constexpr int FT = BIAS == BIAS_NONE ? 2 * TN : OT == OUT_F32 ? 2 : 4, first = decltype(group_tag)::value * FT;
            if constexpr (first < 2 * TN) {
                if constexpr (BIAS != BIAS_NONE) {
#pragma unroll
                    for (int t = 0; t < FT; ++t) scale[first + t].load_bias8(p, min(cn0 + wn * WTN + (first + t) * 16 + half * 8, p.N - 8));
                    TG_FENCE();
                }
                // (one call per row group instead of a loop, see fp8_gemm_tile256.h)
                auto rows = [&](auto tm_tag) __attribute__((always_inline)) {
                    constexpr int tm = decltype(tm_tag)::value;
#pragma unroll
                    for (int t = first; t < first + FT; ++t) {
                        const int col = cn0 + wn * WTN + t * 16 + half * 8;
                        v4f x, y;
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            x[r] = scale[t].finished(read_acc(acc[t / 2][tm][8 * (t & 1) + r]), srow[tm], r);
                            y[r] = scale[t].finished(read_acc(acc[t / 2][tm][8 * (t & 1) + 4 + r]), srow[tm], 4 + r);
                        }
                        out.template put8<OT>(col < p.N ? dsts[tm] + (uint32_t)col * SIZE : kBeyond, x, y);
                        TG_FENCE();
                    }
                };
                rows(std::integral_constant<int, 0>{}); rows(std::integral_constant<int, 1>{});
                rows(std::integral_constant<int, 2>{}); rows(std::integral_constant<int, 3>{});
            }
        };
        group(std::integral_constant<int, 0>{});
        group(std::integral_constant<int, 1>{});
        group(std::integral_constant<int, 2>{});
        group(std::integral_constant<int, 3>{});
        if (!more) break;
#pragma unroll
        for (int tn = 0; tn < TN; ++tn)
#pragma unroll
            for (int tm = 0; tm < TM; ++tm) acc[tn][tm] = 0;
    }
#undef TG_FENCE
    __builtin_amdgcn_s_waitcnt(kWaitAll);  // the re-fetches past the end must land before the workgroup's LDS is released
#endif
}

}  // namespace tg
