// Tiles of 32 x 64 to 256 x 128 of a product in 8-bit integers over a ring of LDS stages, for the row counts between decoding and those that
// fill whole rounds of 256 x 256 tiles, and for the segments of rows that belong to experts: the schedule of fp8_gemm_tile_ring.h over int8 MFMAs.
//
// One workgroup per compute unit: four waves compute (2 x 2), four waves only request the next K steps' slabs by direct global->LDS loads; one
// barrier per step, in front of its last column tiles.  The reasons stand in fp8_gemm_tile_ring.h.  What differs:
//   * a K step of 128 bytes is two 16x16x64 MFMAs per output, issued a row group apart, so that none waits for the other.  (Four 32x32x32 ones, at a
//     higher rate, are ahead by up to 10 % while few compute units work, as 256 x 4096 x 4096 in 192 x 128 tiles 19.8 -> 18.2 us, and behind by 5 to 7 % on a full chip,
//     where power counts: 1400 x 12288 x 5120 in 192 x 192 tiles 80.0 -> 85.9, 2048 x 4096 x 4096 in 256 x 128 32.4 -> 35.5.  Where the chip is not full smaller
//     tiles are chosen, whose steps are loads.)
//   * the scales and biases of a tile come to LDS while its first steps are on their way;
//   * a tile's descriptors start at its own first rows, so that operands may be of any size and a ragged tile's rows anywhere;
//   * K is any multiple of 16: chunks of the last step behind a row's end are requested from beyond the descriptor's range, which makes them
//     zeros in LDS;
//   * partial sums of a split K are int32, and their sum is exact.
// Small tiles are bound inside their compute unit: a step of 64 x 128 takes some 580 cycles with 240 workgroups and 680 with four, so it does not wait for a shared L2.
// The MFMAs are busy 256 of them, fragment reads hold the LDS port for 195, and 24 KB are filled beside these.  333 x 5120 x 12288 takes 30 us (1.37 POP/s).
#pragma once

#include "int8_device.h"

namespace tg {

#define TG_FENCE() __builtin_amdgcn_sched_barrier(0)

// A computing wave's part of a tile: its accumulators and fragments, in which order they are multiplied and refilled, and which outputs an accumulator
// register is.
template <int TM, int TN>
struct RingPart {
    static constexpr int VECS = TN / 2;  // vectors of eight columns that a lane has of a row
    static constexpr int WS = TN == 6 ? 3 : 4, LAST = TN == 4 ? 2 : 1;  // weight fragment sets, column tiles behind the barrier
    static_assert(TN == 2 || TN == 4 || TN == 6, "column tiles");
    v4i acc[TN][TM];
    v8i af[TM], wf[WS];
    uint32_t frag0, wfrag0;
    int li, lg;
    __device__ __forceinline__ void init(int lane, int row0, int col0, int b_base) {
        li = lane & 15, lg = lane >> 4;
        frag0 = (row0 + li) * kKBlock + ((lg ^ swz16(li)) << 4);
        const int wrow = ((li >> 2) << 3) | (li & 3);
        wfrag0 = b_base + (col0 + wrow) * kKBlock + ((lg ^ swz_w(wrow)) << 4);
        clear();
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int tn = 0; tn < TN; ++tn)
#pragma unroll
            for (int tm = 0; tm < TM; ++tm) acc[tn][tm] = v4i{0, 0, 0, 0};
    }
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
        // (in the K loop's order: the compiler waits at its top for what is needed on either way in)
        read_w(0, base);
        if constexpr (TN > 2) read_w(1, base);
        TG_FENCE();
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) {
            read_a<WGM>(tm, base);
            TG_FENCE();
        }
        if constexpr (TN == 2) read_w(1, base);
    }
    // column tile by column tile: all row groups' first halves, then the second ones
    // (PARTIAL: the upper half of the row groups only where it holds rows, see the kernel over experts)
    template <bool PARTIAL>
    __device__ __forceinline__ void before(const uint8_t* cur, bool upper) {
#pragma unroll
        for (int tn = 0; tn < TN - LAST; ++tn) {
            constexpr int H = PARTIAL ? (TM + 1) / 2 : TM;
#pragma unroll
            for (int tm = 0; tm < H; ++tm) {
                acc[tn][tm] = mfma_i8(lo4(wf[tn % WS]), lo4(af[tm]), acc[tn][tm]);
                if (tm == 0 && tn + 2 < TN) read_w(tn + 2, cur);
                TG_FENCE();
            }
#pragma unroll
            for (int tm = 0; tm < H; ++tm) acc[tn][tm] = mfma_i8(hi4(wf[tn % WS]), hi4(af[tm]), acc[tn][tm]);
            TG_FENCE();
            if (H < TM && upper) {
#pragma unroll
                for (int tm = H; tm < TM; ++tm) acc[tn][tm] = mfma_i8(lo4(wf[tn % WS]), lo4(af[tm]), acc[tn][tm]);
#pragma unroll
                for (int tm = H; tm < TM; ++tm) acc[tn][tm] = mfma_i8(hi4(wf[tn % WS]), hi4(af[tm]), acc[tn][tm]);
                TG_FENCE();
            }
        }
    }
    // row group by row group: the last MFMA of one releases its fragment
    template <int WGM, bool PARTIAL>
    __device__ __forceinline__ void behind(const uint8_t* nxt, bool upper) {
        constexpr int H = PARTIAL ? (TM + 1) / 2 : TM;
        read_w(0, nxt);
        if constexpr (TN > 2) read_w(1, nxt);
        TG_FENCE();
        groups<WGM, 0, H>(nxt);
        if (H < TM && upper) groups<WGM, H, TM>(nxt);
        if constexpr (TN == 2) read_w(1, nxt);  // (its registers were the last MFMAs')
    }
    template <int WGM, int FROM, int TO>
    __device__ __forceinline__ void groups(const uint8_t* nxt) {
#pragma unroll
        for (int tm = FROM; tm < TO; ++tm) {
#pragma unroll
            for (int tn = TN - LAST; tn < TN; ++tn) acc[tn][tm] = mfma_i8(lo4(wf[tn % WS]), lo4(af[tm]), acc[tn][tm]);
#pragma unroll
            for (int tn = TN - LAST; tn < TN; ++tn) acc[tn][tm] = mfma_i8(hi4(wf[tn % WS]), hi4(af[tm]), acc[tn][tm]);
            TG_FENCE();
            read_a<WGM>(tm, nxt);
            TG_FENCE();
        }
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

// A loading wave's share of a tile's slabs, and its requests.
template <int BM, int BN, int NL>
struct RingLoader {
    static constexpr int A_IT = BM / (8 * NL), B_IT = BN / (8 * NL), STAGE_BYTES = (BM + BN) * kKBlock;
    static constexpr uint32_t kOutOfRange = 0x80000000u;  // beyond the descriptor's 2^31 - 1 bytes
    uint32_t a_off[A_IT], b_off[B_IT], lds0;
    v4i rsrc_a, rsrc_b;
    int lw, lrow, lj, ljb;
    __device__ __forceinline__ void init(int wave, int lane, uint32_t lds) {
        lw = wave, lrow = lane >> 3;
        lj = (lane & 7) ^ swz16(lrow);
        ljb = (lane & 7) ^ swz_w(((lw & 1) << 3) | lrow);
        lds0 = lds + lw * 1024;
    }
    __device__ __forceinline__ void set(const Int8GemmParams& p, int64_t m0, int n0, int rows_valid, int expert) {
#pragma unroll
        for (int i = 0; i < A_IT; ++i) a_off[i] = (uint32_t)min((i * NL + lw) * 8 + lrow, rows_valid - 1) * (uint32_t)p.K + lj * 16;
#pragma unroll
        for (int i = 0; i < B_IT; ++i) b_off[i] = (uint32_t)min((i * NL + lw) * 8 + lrow, p.N - 1 - n0) * (uint32_t)p.K + ljb * 16;
        rsrc_a = make_rsrc(p.A + m0 * p.K), rsrc_b = make_rsrc(p.B + ((int64_t)expert * p.N + n0) * p.K);
    }
    __device__ __forceinline__ void issue(int K, int kstep, int stage) const {
        const int k0 = kstep * kKBlock;
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
    }
};

// The wave's part of the tile at (m0, n0), finished and stored: its columns from col_in on, its row groups interleaved with the other waves'.
template <int TM, int TN, int WGM, bool BIAS>
__device__ __forceinline__ void ring_store(const Int8GemmParams& p, const RingPart<TM, TN>& part, int64_t m0, int n0, int rows_valid, int wm, int col_in,
                                           const float* s_row, const float* s_col, const float* s_bias) {
    constexpr int VECS = RingPart<TM, TN>::VECS;
    const int li = part.row();
    auto emit_whole = [&](auto type_tag) __attribute__((always_inline)) {
        constexpr int OT = decltype(type_tag)::value;
        constexpr int FV = VECS % 2 == 0 ? 2 : VECS; // vectors whose factors are in registers at a time
        static_assert(VECS % FV == 0, "whole groups of them");
#pragma unroll
        for (int v0 = 0; v0 < VECS; v0 += FV) {
            float f[FV][8], b[FV][8];
#pragma unroll
            for (int v = 0; v < FV; ++v)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int at = col_in + part.column(v0 + v) + i;
                    f[v][i] = s_col[at];
                    b[v][i] = BIAS ? s_bias[at] : kNoBias;
                }
#pragma unroll
            for (int tm = 0; tm < TM; ++tm) {
                const int rt = (tm * WGM + wm) * 16 + li;
                if (rt >= rows_valid) continue;
                const float sa = s_row[rt];
#pragma unroll
                for (int v = 0; v < FV; ++v) {
                    const int col = n0 + col_in + part.column(v0 + v);
                    if (col >= p.N) continue;
                    v4f x, y;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        x[r] = finish(part.get(v0 + v, tm, r), sa, f[v][r], b[v][r]);
                        y[r] = finish(part.get(v0 + v, tm, 4 + r), sa, f[v][4 + r], b[v][4 + r]);
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
    for (int tm = 0; tm < TM; ++tm) {
        const int rt = (tm * WGM + wm) * 16 + li;
        if (rt >= rows_valid) continue;
        const float sa = s_row[rt];
#pragma unroll
        for (int v = 0; v < VECS; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int at = col_in + part.column(v) + i;
                if (n0 + at < p.N) put1(p, (m0 + rt) * p.ldc + n0 + at, finish(part.get(v, tm, i), sa, s_col[at], BIAS ? s_bias[at] : kNoBias));
            }
    }
}

template <int BM, int BN, int STAGES, bool SPLIT>
__global__ void __launch_bounds__(512, 1) int8_gemm_ring_kernel(const Int8GemmParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int NL = 4, WGN = BN == 32 ? 1 : 2, WGM = 4 / WGN;
    constexpr int WTN = BN / WGN;
    constexpr int TM = BM / (16 * WGM), TN = WTN / 16;
    using Part = RingPart<TM, TN>;
    constexpr int VECS = Part::VECS;
    constexpr int A_IT = BM / (8 * NL), B_IT = BN / (8 * NL);
    constexpr int STAGE_BYTES = (BM + BN) * kKBlock;
    constexpr int PER_STEP = A_IT + B_IT;
    constexpr int FACTORS = (BM + 2 * BN) * 4;
    static_assert(BM % (16 * WGM) == 0 && STAGES >= 3 && STAGES * STAGE_BYTES + FACTORS <= 160 * 1024, "shape");

    __shared__ __align__(1024) uint8_t lds[STAGES * STAGE_BYTES];  // stage s: A slab, then B slab
    // scales of the tile's rows, scales and biases of its columns: brought here while the first steps are on their way
    __shared__ __align__(16) float s_row[BM], s_col[BN], s_bias[BN];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int K = p.K;
    const int tiles_n = (p.N + BN - 1) / BN;
    const int tiles_m = (p.M + BM - 1) / BM;
    const int pid = xcd_remap((int)blockIdx.x, tiles_m * tiles_n);
    constexpr int GM = 8;
    const int width = GM * tiles_n;
    const int group = pid / width, first_m = group * GM;
    const int gsz = min(tiles_m - first_m, GM);
    const int64_t m0 = (int64_t)(first_m + (pid % width) % gsz) * BM;
    const int n0 = ((pid % width) / gsz) * BN;
    const int rows_valid = (int)min((int64_t)BM, p.M - m0);
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
        RingLoader<BM, BN, NL> loader;
        loader.init(wave - 4, lane, lds_address(lds));
        loader.set(p, m0, n0, rows_valid, 0);
        // Where a weight row is read once, workgroups start at different K steps and go round: rows a power of two apart would meet on few memory
        // channels (128 x 28672 x 4096 in 128 x 128 tiles 32.8 -> 28.7 us; with eight row tiles, 1024 x 8192 x 8192 in 256 x 128, 57 -> 63).
        const int rot = tiles_m == 1 ? (int)((blockIdx.x >> 3) % (unsigned)nsteps) : 0;
        auto issue = [&](int kstep, int stage) {
            const int at = min(kstep, last) + rot;
            loader.issue(K, at < ks_end ? at : at - nsteps, stage);
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
    Part part;
    part.init(lane, wm * 16, wn * WTN, BM * kKBlock);
    const int li = part.row();

    if constexpr (!SPLIT) {
        for (int i = tid; i < BM; i += 256) s_row[i] = p.sa[(m0 + min(i, rows_valid - 1)) * p.sa_step];
        for (int i = tid; i < BN; i += 256) {
            const int col = min(n0 + i, p.N - 1);
            s_col[i] = p.sb[(int64_t)col * p.sb_step];
            s_bias[i] = load_bias(p.bias, p.bias_type, col);
        }
    }
    __builtin_amdgcn_s_waitcnt(kWaitLds);  // (and no scalar load is under way in the K loop: the compiler would wait for all reads of LDS at its top)
    __builtin_amdgcn_s_barrier();  // step 0 has landed
    part.template first<WGM>(lds);
    int stage = 0;
    for (int k = 0; k < nsteps; ++k) {
        const uint8_t* cur = lds + stage * STAGE_BYTES;
        stage = stage == STAGES - 1 ? 0 : stage + 1;
        const uint8_t* nxt = lds + stage * STAGE_BYTES;
        TG_FENCE();
        part.template before<false>(cur, true);
        __builtin_amdgcn_s_waitcnt(kWaitLds);  // all my reads of step k are done
        __builtin_amdgcn_s_barrier();          // step k+1 is visible
        TG_FENCE();
        part.template behind<WGM, false>(nxt, true);
    }
    part.keep();

    const int col0 = n0 + wn * WTN;
    if constexpr (SPLIT) {
        int* mine = p.partials + (int64_t)blockIdx.y * p.M * p.N;
#pragma unroll
        for (int tm = 0; tm < TM; ++tm) {
            const int rt = (tm * WGM + wm) * 16 + li;
            if (rt >= rows_valid) continue;
#pragma unroll
            for (int v = 0; v < VECS; ++v) {
                const int col = col0 + part.column(v);
                int* to = mine + (m0 + rt) * p.N + col;
                if (p.N % 8 == 0) {
                    if (col >= p.N) continue;
                    *reinterpret_cast<v4i*>(to) = v4i{part.get(v, tm, 0), part.get(v, tm, 1), part.get(v, tm, 2), part.get(v, tm, 3)};
                    *reinterpret_cast<v4i*>(to + 4) = v4i{part.get(v, tm, 4), part.get(v, tm, 5), part.get(v, tm, 6), part.get(v, tm, 7)};
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (col + i < p.N) to[i] = part.get(v, tm, i);
                }
            }
        }
        return;
    }
    ring_store<TM, TN, WGM, true>(p, part, m0, n0, rows_valid, wm, wn * WTN, s_row, s_col, s_bias);
#endif
}

// The same over the segments of rows that belong to experts, persistent: a workgroup walks tiles b, b + grid, ... of the experts' row tiles x column tiles, and
// its loading waves run on into the next tile while the others store one.  24576 rows over 64 experts of (2816, 2048) in 192 x 192 tiles: 189 us, launched tile by tile
// 210; 6000 rows in 160 x 192: 93, 97 (4.1 TB/s of weights, rows and outputs).
template <int BM, int BN, int STAGES>
__global__ void __launch_bounds__(512, 1) int8_gemm_ring_experts_kernel(const Int8GemmParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int NL = 4, WGN = BN == 32 ? 1 : 2, WGM = 4 / WGN;
    constexpr int WTN = BN / WGN;
    constexpr int TM = BM / (16 * WGM), TN = WTN / 16;
    using Loader = RingLoader<BM, BN, NL>;
    constexpr int PER_STEP = Loader::A_IT + Loader::B_IT, FACTORS = BM + BN;
    static_assert(BM <= 256 && BN <= 256 && STAGES * Loader::STAGE_BYTES + 2 * FACTORS * 4 <= 160 * 1024, "shape");
    constexpr int kPro = (STAGES - 1) * PER_STEP, kLoop = (STAGES - 2) * PER_STEP;  // loads that may stay in flight
    constexpr int kWaitPro = 0x0F70 | (kPro & 15) | ((kPro >> 4) << 14);
    constexpr int kWaitLoop = 0x0F70 | (kLoop & 15) | ((kLoop >> 4) << 14);
    constexpr int kWaitAll = 0x0F70;
    constexpr int kWaitLds = 0xC07F;

    __shared__ __align__(1024) uint8_t lds[STAGES * Loader::STAGE_BYTES];
    __shared__ __align__(16) float factors[2][FACTORS];  // scales of a tile's rows, then of its columns; the next tile's beside them

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int tiles_n = (p.N + BN - 1) / BN, grid = (int)gridDim.x;
    RaggedWalk<BM> walk;
    const int total = walk.start(p, lane, tiles_n);
    int v = (int)blockIdx.x;
    if (v >= total) return;
    const int tiles = (total - v + grid - 1) / grid, nsteps = (p.K + kKBlock - 1) / kKBlock;
    int expert, m0, rows_valid, tile_n;

    if (wave >= 4) {
        Loader loader;
        loader.init(wave - 4, lane, lds_address(lds));
        int left = tiles, k = 0;
        auto go = [&]() {
            walk.find(p, lane, xcd_remap(v, total), tiles_n, expert, m0, rows_valid, tile_n);
            loader.set(p, m0, tile_n * BN, rows_valid, expert);
            v += grid;
        };
        go();
        auto issue = [&](int stage) {
            loader.issue(p.K, k, stage);
            if (k + 1 < nsteps) {
                ++k;
            } else if (left > 1) {  // (behind the last tile's last step: that one again)
                --left;
                k = 0;
                go();
            }
        };
#pragma unroll
        for (int s = 0; s < STAGES; ++s) issue(s);
        __builtin_amdgcn_s_waitcnt(kWaitPro);
        __builtin_amdgcn_s_barrier();
        int stage = 0;
        for (int64_t s = 0; s < (int64_t)tiles * nsteps; ++s) {
            __builtin_amdgcn_s_waitcnt(kWaitLoop);
            __builtin_amdgcn_s_barrier();
            issue(stage);
            stage = stage == STAGES - 1 ? 0 : stage + 1;
        }
        __builtin_amdgcn_s_waitcnt(kWaitAll);
        return;
    }

    const int wm = wave % WGM, wn = wave / WGM;
    RingPart<TM, TN> part;
    part.init(lane, wm * 16, wn * WTN, BM * kKBlock);
    __builtin_amdgcn_s_waitcnt(kWaitLds);
    __builtin_amdgcn_s_barrier();  // step 0 has landed
    int stage = 0;
    for (int t = 0; t < tiles; ++t) {
        walk.find(p, lane, xcd_remap(v, total), tiles_n, expert, m0, rows_valid, tile_n);
        v += grid;
        const int n0 = tile_n * BN;
        // asked for here, in LDS from the tile's last step on
        const float row = p.sa[((int64_t)m0 + min(tid, rows_valid - 1)) * p.sa_step];
        const float col = p.sb[((int64_t)expert * p.N + min(n0 + tid, p.N - 1)) * p.sb_step];
        float* const scales = factors[t & 1];
        // An expert's last rows may leave the upper half of the row groups empty: then its MFMAs and fragments are left out (6000 rows, 1 to 711 an expert, in 192 x 192 tiles
        // 101 -> 99 us; in steps of two groups no better).
        const bool upper = rows_valid > (TM + 1) / 2 * 16 * WGM;
        // (again behind the first tile: fragments that lived through the stores would be more than the registers hold)
        part.template first<WGM>(lds + stage * Loader::STAGE_BYTES);
        for (int k = 0; k < nsteps; ++k) {
            if (k == nsteps - 1) {
                if (tid < BM) scales[tid] = row;
                if (tid < BN) scales[BM + tid] = col;
            }
            const uint8_t* cur = lds + stage * Loader::STAGE_BYTES;
            stage = stage == STAGES - 1 ? 0 : stage + 1;
            const uint8_t* nxt = lds + stage * Loader::STAGE_BYTES;
            TG_FENCE();
            part.template before<true>(cur, upper);
            __builtin_amdgcn_s_waitcnt(kWaitLds);
            __builtin_amdgcn_s_barrier();
            TG_FENCE();
            part.template behind<WGM, true>(nxt, upper);
        }
        part.keep();
        // (as if written here: what the stores compute from them would be held through all K loops)
        asm volatile("" : "+v"(part.li), "+v"(part.lg));
        ring_store<TM, TN, WGM, false>(p, part, m0, n0, rows_valid, wm, wn * WTN, scales, scales + BM, nullptr);
        part.clear();
    }
#endif
}

template <int BM, int BN, int STAGES>
inline hipError_t launch_int8_ring(const Int8GemmParams& p, hipStream_t stream) {
    const int64_t cols = ((int64_t)p.N + BN - 1) / BN;
    const int64_t tiles = cols * (p.m_indptr ? most_row_tiles(p.M, p.E, BM) : ((int64_t)p.M + BM - 1) / BM);
    if (p.m_indptr) {
        if (tiles > INT32_MAX / 2) return hipErrorInvalidValue;
        hipLaunchKernelGGL((int8_gemm_ring_experts_kernel<BM, BN, STAGES>), dim3((unsigned)walking_grid(tiles, compute_units())), dim3(512), 0, stream, p);
        return hipGetLastError();
    }
    if (tiles * p.split_k * 512 > kMostThreads) return hipErrorInvalidValue;
    const dim3 grid((unsigned)tiles, p.split_k), block(512);
    if (p.split_k > 1) hipLaunchKernelGGL((int8_gemm_ring_kernel<BM, BN, STAGES, true>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((int8_gemm_ring_kernel<BM, BN, STAGES, false>), grid, block, 0, stream, p);
    return hipGetLastError();
}

#undef TG_FENCE

}  // namespace tg
