// 256 x 256 tiles of a product in 8-bit integers, persistent, with a hand-ordered K loop (prompts): the schedule of fp8_gemm_tile256.h over
// int8 MFMAs.
//
// Four waves, one per SIMD, each with a 128 x 128 part of the tile, one workgroup per compute unit that walks tiles b, b + grid, ... of the rastered
// sequence; two activation slabs and three weight slabs (160 KiB, all of LDS); requests two steps ahead, running on into the next tile; one barrier per
// step in front of its last sixteen outputs.  The reasons stand in fp8_gemm_tile256.h.  What differs: a K step of 128 bytes is two MFMAs of 64 per
// output, issued four outputs apart so that none waits for the other, and the epilogue has a scale per row and per column and a bias.
// K must be a multiple of 128 and at least 256, the operands below 2 GiB each, the outputs in whole vectors (vec_store).
#pragma once

#include "int8_device.h"

namespace tg {

__global__ void __launch_bounds__(256, 1) int8_gemm_tile256_kernel(const Int8GemmParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int BM = 256, BN = 256, WGM = 2, WGN = 2, NW = 4;
    constexpr int WTN = BN / WGN;
    constexpr int TM = 8, TN = WTN / 16;
    constexpr int SLAB = 256 * kKBlock;
    constexpr int A_STAGES = 2, B_STAGES = 3;
    constexpr int IT = 256 / (8 * NW);
    static_assert(TN == 8 && IT == 8, "schedule below is written for 8 x 8 MFMA tiles and 8 + 8 loads per wave");

    __shared__ __align__(1024) uint8_t sA[A_STAGES * SLAB];
    __shared__ __align__(1024) uint8_t sB[B_STAGES * SLAB];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave % WGM, wn = wave / WGM;
    const int K = p.K;
    const int tiles_n = (p.N + BN - 1) / BN, tiles_m = (p.M + BM - 1) / BM;
    const int total = tiles_m * tiles_n, stride = (int)gridDim.x;
    auto origin = [&](int v, int& om0, int& on0) {
        const int pid = xcd_remap(v, total);
        constexpr int GM = 8;
        const int width = GM * tiles_n;
        const int group = pid / width, first_m = group * GM;
        const int gsz = min(tiles_m - first_m, GM);
        om0 = (first_m + (pid % width) % gsz) * BM;
        on0 = ((pid % width) / gsz) * BN;
    };
    int vt = (int)blockIdx.x;
    int m0, n0;
    origin(vt, m0, n0);
    const int nsteps = K / kKBlock, last = nsteps - 1;

    const int lrow = lane >> 3;
    const int lj = (lane & 7) ^ swz16(lrow);
    const int ljb = (lane & 7) ^ swz_w(((wave & 1) << 3) | lrow);
    uint32_t a_off[IT], b_off[IT];
    auto set_offsets = [&](int om0, int on0) {
        const int rv = min(BM, p.M - om0);
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int r = (i * NW + wave) * 8 + lrow;
            a_off[i] = (uint32_t)(om0 + min(r, rv - 1)) * (uint32_t)K + lj * 16;
            b_off[i] = (uint32_t)min(on0 + r, p.N - 1) * (uint32_t)K + ljb * 16;
        }
    };
    set_offsets(m0, n0);
    const v4i rsrc_a = make_rsrc(p.A), rsrc_b = make_rsrc(p.B);
    const uint32_t ldsA = settle(lds_address(sA) + wave * 1024), ldsB = settle(lds_address(sB) + wave * 1024);
    auto load_a = [&](int i, int kstep, int stage) {
        direct_load_b128_settled(rsrc_a, ldsA + stage * SLAB + i * NW * 1024, a_off[i], kstep * kKBlock);
    };
    auto load_b = [&](int i, int kstep, int stage) {
        direct_load_b128_settled(rsrc_b, ldsB + stage * SLAB + i * NW * 1024, b_off[i], kstep * kKBlock);
    };

    const int li = lane & 15, lg = lane >> 4;
    const uint32_t frag0 = wm * 16 * kKBlock + li * kKBlock + ((lg ^ swz16(li)) << 4), frag1 = frag0 ^ 64;
    const int wrow = ((li >> 2) << 3) | (li & 3);
    const uint32_t wfrag0 = wn * WTN * kKBlock + wrow * kKBlock + ((lg ^ swz_w(wrow)) << 4), wfrag1 = wfrag0 ^ 64;
    auto read_a = [&](int tm, const uint8_t* cA) {
        const uint8_t* base = cA + tm * (WGM * 16 * kKBlock);
        return join(*reinterpret_cast<const v4i*>(base + frag0), *reinterpret_cast<const v4i*>(base + frag1));
    };
    auto read_w = [&](int tn, const uint8_t* cB) {
        const uint8_t* base = cB + ((tn >> 1) * 32 + (tn & 1) * 4) * kKBlock;
        return join(*reinterpret_cast<const v4i*>(base + wfrag0), *reinterpret_cast<const v4i*>(base + wfrag1));
    };

    v4i acc[TN][TM];
#pragma unroll
    for (int tn = 0; tn < TN; ++tn)
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) acc[tn][tm] = v4i{0, 0, 0, 0};

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
    v8i af[TM], wf[4];
    wf[0] = read_w(0, sB);
    wf[1] = read_w(1, sB);
#pragma unroll
    for (int tm = 0; tm < TM; ++tm) af[tm] = read_a(tm, sA);

    int sa = 0, sb = 0;
    for (;;) {
        const int cm0 = m0, cn0 = n0;
        bool more = false;
        for (int k = 0; k < nsteps; ++k) {
            if (k == nsteps - 2) {
                more = vt + stride < total;
                if (more) {
                    vt += stride;
                    origin(vt, m0, n0);
                    set_offsets(m0, n0);
                }
            }
            int k2 = k + 2;
            if (k2 >= nsteps) k2 = more ? k2 - nsteps : last;
            const int sa1 = sa ^ 1;
            const int sb1 = sb == B_STAGES - 1 ? 0 : sb + 1;
            const int sb2 = sb1 == B_STAGES - 1 ? 0 : sb1 + 1;
            const uint8_t* cB = sB + sb * SLAB;
            TG_FENCE();
            // column tiles 0 .. 5 in halves of four outputs (eight MFMAs); behind each half of the first four a direct load, behind each first
            // half the weight fragment of the column tile after next
#pragma unroll
            for (int tn = 0; tn < 6; ++tn) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[tn][4 * h + j] = mfma_i8(lo4(wf[tn & 3]), lo4(af[4 * h + j]), acc[tn][4 * h + j]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[tn][4 * h + j] = mfma_i8(hi4(wf[tn & 3]), hi4(af[4 * h + j]), acc[tn][4 * h + j]);
                    TG_FENCE();
                    if (2 * tn + h < IT) load_b(2 * tn + h, k2, sb2);
                    if (h == 0) wf[(tn + 2) & 3] = read_w(tn + 2, cB);
                    TG_FENCE();
                }
            }
            __builtin_amdgcn_s_waitcnt(kWaitBut8);
            __builtin_amdgcn_s_waitcnt(kWaitLds);
            __builtin_amdgcn_s_barrier();
            TG_FENCE();
            const uint8_t* nA = sA + sa1 * SLAB;
            const uint8_t* nB = sB + sb1 * SLAB;
            wf[0] = read_w(0, nB);
            wf[1] = read_w(1, nB);
            TG_FENCE();
#pragma unroll
            for (int tm = 0; tm < TM; ++tm) {
                acc[6][tm] = mfma_i8(lo4(wf[2]), lo4(af[tm]), acc[6][tm]);
                acc[7][tm] = mfma_i8(lo4(wf[3]), lo4(af[tm]), acc[7][tm]);
                acc[6][tm] = mfma_i8(hi4(wf[2]), hi4(af[tm]), acc[6][tm]);
                acc[7][tm] = mfma_i8(hi4(wf[3]), hi4(af[tm]), acc[7][tm]);
                TG_FENCE();
                af[tm] = read_a(tm, nA);
                load_a(tm, k2, sa);
                TG_FENCE();
            }
            sa = sa1;
            sb = sb1;
        }
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) asm volatile("" : : "v"(af[tm]));
        asm volatile("" : : "v"(wf[0]), "v"(wf[1]));

        // ---- epilogue, straight from the accumulators
        const int rows_valid = min(BM, p.M - cm0);
        int dsts[TM];
        float srow[TM];
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) {
            const int rt = (tm * WGM + wm) * 16 + li;
            dsts[tm] = rt < rows_valid ? cm0 + rt : -1;
            srow[tm] = p.sa[(int64_t)(cm0 + min(rt, rows_valid - 1)) * p.sa_step];
        }
        // two pairs of column tiles at a time: their 64 columns are whole lines of a 16-bit output, and their factors half of the registers
        auto emit = [&](auto type_tag) __attribute__((always_inline)) {
            constexpr int OT = decltype(type_tag)::value;
            auto half = [&](auto half_tag) __attribute__((always_inline)) {
                constexpr int first = decltype(half_tag)::value * 2;
                ColumnFactors f[2];
                int cols[2];
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    cols[t] = cn0 + wn * WTN + (first + t) * 32 + lg * 8;
                    f[t].load(p, p.sb, min(cols[t], p.N - 8));
                }
                // (one call per row group instead of a loop, see fp8_gemm_tile256.h)
                auto rows = [&](auto tm_tag) __attribute__((always_inline)) {
                    constexpr int tm = decltype(tm_tag)::value;
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (dsts[tm] < 0 || cols[t] >= p.N) continue;
                        v4f x, y;
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            x[r] = finish(acc[2 * (first + t)][tm][r], srow[tm], f[t].s[r], f[t].b[r]);
                            y[r] = finish(acc[2 * (first + t) + 1][tm][r], srow[tm], f[t].s[4 + r], f[t].b[4 + r]);
                        }
                        put8<OT>(p.C, (int64_t)dsts[tm] * p.ldc + cols[t], x, y);
                    }
                };
                rows(std::integral_constant<int, 0>{}); rows(std::integral_constant<int, 1>{});
                rows(std::integral_constant<int, 2>{}); rows(std::integral_constant<int, 3>{});
                rows(std::integral_constant<int, 4>{}); rows(std::integral_constant<int, 5>{});
                rows(std::integral_constant<int, 6>{}); rows(std::integral_constant<int, 7>{});
            };
            half(std::integral_constant<int, 0>{});
            half(std::integral_constant<int, 1>{});
        };
        if (p.out_type == OUT_BF16) emit(std::integral_constant<int, OUT_BF16>{});
        else if (p.out_type == OUT_F32) emit(std::integral_constant<int, OUT_F32>{});
        else emit(std::integral_constant<int, OUT_F16>{});
        if (!more) break;
#pragma unroll
        for (int tn = 0; tn < TN; ++tn)
#pragma unroll
            for (int tm = 0; tm < TM; ++tm) acc[tn][tm] = v4i{0, 0, 0, 0};
    }
#undef TG_FENCE
    __builtin_amdgcn_s_waitcnt(kWaitAll);  // the re-fetches past the end must land before the workgroup's LDS is released
#endif
}

}  // namespace tg
