// Tiles of 32 x 64 to 256 x 128 of a product in 8-bit integers over a ring of LDS stages, for the row counts between decoding and those that
// fill whole rounds of 256 x 256 tiles, and for the segments of rows that belong to experts: the schedule of fp8_gemm_tile_ring.h over int8 MFMAs.
//
// One workgroup per compute unit: four waves compute (2 x 2), four waves only request the next K steps' slabs by direct global->LDS loads; one
// barrier per step, in front of its last column tiles.  The reasons stand in fp8_gemm_tile_ring.h.  What differs:
//   * a K step of 128 bytes is two MFMAs of 64 per output; the two are issued a row group apart, so that none waits for the other;
//   * a tile's descriptors start at its own first rows, so that operands may be of any size and a ragged tile's rows anywhere;
//   * K is any multiple of 16: chunks of the last step behind a row's end are requested from beyond the descriptor's range, which makes them
//     zeros in LDS;
//   * partial sums of a split K are int32, and their sum is exact.
#pragma once

#include "int8_device.h"

namespace tg {

template <int BM, int BN, int STAGES, bool SPLIT, bool RAGGED>
__global__ void __launch_bounds__(512, 1) int8_gemm_ring_kernel(const Int8GemmParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int NL = 4, WGN = BN == 32 ? 1 : 2, WGM = 4 / WGN;
    constexpr int WTN = BN / WGN;
    constexpr int TM = BM / (16 * WGM), TN = WTN / 16;
    constexpr int A_IT = BM / (8 * NL), B_IT = BN / (8 * NL);
    constexpr int STAGE_BYTES = (BM + BN) * kKBlock;
    constexpr int PER_STEP = A_IT + B_IT;
    constexpr int WS = TN == 6 ? 3 : 4;                 // weight fragment sets
    constexpr int LAST = TN == 4 ? 2 : 1;               // column tiles behind the barrier
    static_assert(BM % (16 * WGM) == 0 && (TN == 2 || TN == 4 || TN == 6) && STAGES >= 3 && STAGES * STAGE_BYTES <= 160 * 1024, "shape");
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
#define TG_FENCE() __builtin_amdgcn_sched_barrier(0)

    if (wave >= 4) {
        // ------------------------------------------------------------ loading waves
        const int lw = wave - 4;
        const int lrow = lane >> 3;
        const int lj = (lane & 7) ^ swz16(lrow);
        const int ljb = (lane & 7) ^ swz_w(((lw & 1) << 3) | lrow);
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
    const int li = lane & 15, lg = lane >> 4;
    const uint32_t frag0 = wm * 16 * kKBlock + li * kKBlock + ((lg ^ swz16(li)) << 4), frag1 = frag0 ^ 64;
    const int wrow = ((li >> 2) << 3) | (li & 3);
    const uint32_t wfrag0 = BM * kKBlock + wn * WTN * kKBlock + wrow * kKBlock + ((lg ^ swz_w(wrow)) << 4), wfrag1 = wfrag0 ^ 64;

    v4i acc[TN][TM];
#pragma unroll
    for (int tn = 0; tn < TN; ++tn)
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) acc[tn][tm] = v4i{0, 0, 0, 0};

    // the scales and biases of this lane's rows and columns, asked for in front of the K loop where there are registers for them
    const float* sb = p.sb + (int64_t)expert * p.N * p.sb_step;
    float srow[TM];
#pragma unroll
    for (int tm = 0; tm < TM; ++tm) srow[tm] = p.sa[(m0 + min((tm * WGM + wm) * 16 + li, rows_valid - 1)) * p.sa_step];

    v8i af[TM], wf[WS];
    auto read_a = [&](int tm, const uint8_t* base) {
        const uint8_t* a = base + tm * (WGM * 16 * kKBlock);
        af[tm] = join(*reinterpret_cast<const v4i*>(a + frag0), *reinterpret_cast<const v4i*>(a + frag1));
    };
    auto read_w = [&](int tn, const uint8_t* base) {
        const uint8_t* b = base + ((tn >> 1) * 32 + (tn & 1) * 4) * kKBlock;
        wf[tn % WS] = join(*reinterpret_cast<const v4i*>(b + wfrag0), *reinterpret_cast<const v4i*>(b + wfrag1));
    };
    __builtin_amdgcn_s_barrier();  // step 0 has landed
    read_w(0, lds);
    read_w(1, lds);
#pragma unroll
    for (int tm = 0; tm < TM; ++tm) read_a(tm, lds);
    int stage = 0;
    for (int k = 0; k < nsteps; ++k) {
        const uint8_t* cur = lds + stage * STAGE_BYTES;
        stage = stage == STAGES - 1 ? 0 : stage + 1;
        const uint8_t* nxt = lds + stage * STAGE_BYTES;
        TG_FENCE();
        // in front of the barrier column tile by column tile: all row groups' first halves, then the second ones
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
        __builtin_amdgcn_s_waitcnt(kWaitLds);  // all my reads of step k are done
        __builtin_amdgcn_s_barrier();          // step k+1 is visible
        TG_FENCE();
        read_w(0, nxt);
        if constexpr (TN > 2) read_w(1, nxt);
        TG_FENCE();
        // behind it row group by row group: the last MFMA of one releases its fragment
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) {
#pragma unroll
            for (int tn = TN - LAST; tn < TN; ++tn) acc[tn][tm] = mfma_i8(lo4(wf[tn % WS]), lo4(af[tm]), acc[tn][tm]);
#pragma unroll
            for (int tn = TN - LAST; tn < TN; ++tn) acc[tn][tm] = mfma_i8(hi4(wf[tn % WS]), hi4(af[tm]), acc[tn][tm]);
            TG_FENCE();
            read_a(tm, nxt);
            TG_FENCE();
        }
        if constexpr (TN == 2) read_w(1, nxt);  // (its registers were the last MFMAs')
    }
#pragma unroll
    for (int tm = 0; tm < TM; ++tm) asm volatile("" : : "v"(af[tm]));
    asm volatile("" : : "v"(wf[0]), "v"(wf[1]));
#undef TG_FENCE

    const int col0 = n0 + wn * WTN + lg * 8;
    if constexpr (SPLIT) {
        int* mine = p.partials + (int64_t)blockIdx.y * p.M * p.N;
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) {
            const int rt = (tm * WGM + wm) * 16 + li;
            if (rt >= rows_valid) continue;
            const int64_t at = (m0 + rt) * p.N + col0;
#pragma unroll
            for (int tp = 0; tp < TN / 2; ++tp) {
                if (p.N % 8 == 0) {
                    if (col0 + tp * 32 >= p.N) continue;
                    *reinterpret_cast<v4i*>(mine + at + tp * 32) = acc[2 * tp][tm];
                    *reinterpret_cast<v4i*>(mine + at + tp * 32 + 4) = acc[2 * tp + 1][tm];
                } else {
#pragma unroll
                    for (int q = 0; q < 8; ++q)
                        if (col0 + tp * 32 + q < p.N) mine[at + tp * 32 + q] = acc[2 * tp + (q >> 2)][tm][q & 3];
                }
            }
        }
        return;
    }
    auto emit_whole = [&](auto type_tag) __attribute__((always_inline)) {
        constexpr int OT = decltype(type_tag)::value;
        ColumnFactors f[TN / 2];
#pragma unroll
        for (int tp = 0; tp < TN / 2; ++tp) f[tp].load(p, sb, min(col0 + tp * 32, p.N - 8));
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) {
            const int rt = (tm * WGM + wm) * 16 + li;
            if (rt >= rows_valid) continue;
#pragma unroll
            for (int tp = 0; tp < TN / 2; ++tp) {
                if (col0 + tp * 32 >= p.N) continue;
                v4f x, y;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    x[r] = finish(acc[2 * tp][tm][r], srow[tm], f[tp].s[r], f[tp].b[r]);
                    y[r] = finish(acc[2 * tp + 1][tm][r], srow[tm], f[tp].s[4 + r], f[tp].b[4 + r]);
                }
                put8<OT>(p.C, (m0 + rt) * p.ldc + col0 + tp * 32, x, y);
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
    for (int tp = 0; tp < TN / 2; ++tp)
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const int col = col0 + tp * 32 + q;
            if (col >= p.N) continue;
            const float s = sb[(int64_t)col * p.sb_step], b = load_bias(p.bias, p.bias_type, col);
#pragma unroll
            for (int tm = 0; tm < TM; ++tm) {
                const int rt = (tm * WGM + wm) * 16 + li;
                if (rt < rows_valid) put1(p, (m0 + rt) * p.ldc + col, finish(acc[2 * tp + (q >> 2)][tm][q & 3], srow[tm], s, b));
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

}  // namespace tg
