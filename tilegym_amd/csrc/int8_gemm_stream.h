// Products in 8-bit integers over up to 16 or 32 rows, bound by reading the weight once: the two-piece wide form of fp8_gemm_stream.h over int8
// MFMAs, for dense rows and for the segments of rows that belong to experts.
//
// A workgroup of four waves has 4 R weight rows (R <= 16, p.wave_rows) over its whole K range, which it works through in pieces of 512 bytes: each wave
// loads its own rows' piece by direct global->LDS loads of whole 512-byte runs, all of them share the activation piece; piece c + 1 is in flight
// while piece c is multiplied, and piece c + 2 is requested as soon as piece c's fragments are in registers.  Workgroup b starts at piece
// b % (pieces) and goes round, so that rows a power of two apart do not meet on few memory channels; the sums are integers, so the order
// changes no bits.  What a wave does not have (rows behind its R, chunks of K behind a row's end) is requested from beyond the descriptor's
// range: no memory request, zeros in LDS.
//
// Bound by HBM: 16 x 6144 x 4096 takes 8.4 us (3.0 TB/s; the launch and the first piece are half of it), 240 rows over 53 of 64 experts of (2816, 2048) 47 to 50 (6.1 to 6.5 TB/s, part of it
// from the cache behind the L2).
//
// Ragged: a grid row per expert for its first 16 rows, which leaves at once where the expert has none, and grid rows past the experts for
// their further rows, 16 at a time.
#pragma once

#include "int8_device.h"

namespace tg {

template <int MT, bool RAGGED>
__global__ void __launch_bounds__(256) int8_gemm_stream_kernel(const Int8GemmParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int NW = 4;
    constexpr int PIECE = 512;                 // bytes of K per piece and row
    constexpr int BUF = 16 * PIECE;            // a wave's weight rows
    constexpr int ABUF = MT * BUF;             // the activation piece
    constexpr int SPC = PIECE / kKBlock;
    constexpr int A_LOADS = 2 * MT;            // per wave and piece
    constexpr uint32_t kOutOfRange = 0x80000000u;
    __shared__ __align__(1024) uint8_t sW[NW * 2 * BUF];
    __shared__ __align__(1024) uint8_t sA[2 * ABUF];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 15, lg = lane >> 4;
    const int K = p.K, N = p.N;
    int expert = 0, rows = p.M;
    int64_t row0 = 0;
    if constexpr (RAGGED) {
        const int further = (int)blockIdx.y - p.E;  // which of the experts' passes behind their first ones; below 0: an expert's first
        int pass = 0;
        expert = blockIdx.y;
        if (further >= 0) {
            int before = 0;
            expert = -1;
            for (int e0 = 0; e0 < p.E; e0 += 64) {
                const int n = e0 + lane < p.E ? ragged_rows(p, e0 + lane) : 0, passes = n > 0 ? (n - 1) / 16 : 0;
                int upto = before + passes;
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) {
                    const int t = __shfl_up(upto - before, d);
                    if (lane >= d) upto += t;
                }
                const unsigned long long hit = __ballot(upto > further);
                if (hit) {
                    const int l = __ffsll((long long)hit) - 1;
                    expert = e0 + l;
                    pass = further - __shfl(upto - passes, l) + 1;
                    break;
                }
                before = __shfl(upto, 63);
            }
            if (expert < 0) return;
        }
        expert = __builtin_amdgcn_readfirstlane(expert);
        rows = __builtin_amdgcn_readfirstlane(ragged_rows(p, expert) - 16 * pass);
        if (rows <= 0) return;
        row0 = (int64_t)__builtin_amdgcn_readfirstlane(p.m_indptr[expert]) + 16 * __builtin_amdgcn_readfirstlane(pass);
    }
    const int rows_a = min(rows, 16 * MT);
    const int R = p.wave_rows;
    const int n_base = (blockIdx.x * NW + wave) * R;
    const int n_end = min(n_base + R, N);
    const int npieces = (K + PIECE - 1) / PIECE;
    int c_begin = 0, c_end = npieces;
    if (!RAGGED && p.split_k > 1) {  // (ksteps_per_split is a multiple of four steps)
        c_begin = blockIdx.y * (p.ksteps_per_split / SPC);
        c_end = min(c_begin + p.ksteps_per_split / SPC, npieces);
    }
    const int n_first = min(n_base, N - 1);  // (a wave behind the last row asks for nothing)
    const v4i rsrc_b = make_rsrc(p.B + ((int64_t)expert * N + n_first) * K), rsrc_a = make_rsrc(p.A + row0 * K);
    const uint32_t my_lds = lds_address(sW) + wave * 2 * BUF, a_lds = lds_address(sA);
    const uint8_t* my_buf = sW + wave * 2 * BUF;

    // lane l of a load: row 2i + l/32, LDS position l%32 of the row's 32 chunks, which holds logical chunk (l%32) ^ (row % 16)
    const int half = lane >> 5, pos = lane & 31;
    const int tail = K - (npieces - 1) * PIECE;  // bytes of the last piece
    uint32_t w_off[8], a_off[A_LOADS];
    uint32_t w_in = 0, a_in = 0;                 // which of the chunks the last piece has
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = 2 * i + half, chunk = pos ^ r;
        w_off[i] = n_base + r < n_end ? (uint32_t)r * (uint32_t)K + (uint32_t)(chunk << 4) : kOutOfRange;
        w_in |= (uint32_t)(chunk * 16 < tail) << i;
    }
#pragma unroll
    for (int i = 0; i < A_LOADS; ++i) {
        const int r = 2 * (wave + i * NW) + half, chunk = pos ^ (r & 15);
        a_off[i] = r < rows_a ? (uint32_t)r * (uint32_t)K + (uint32_t)(chunk << 4) : kOutOfRange;
        a_in |= (uint32_t)(chunk * 16 < tail) << i;
    }
    auto issue = [&](int c, int buf) {
        const int k0 = c * PIECE;
        if (c == npieces - 1 && tail != PIECE) {
#pragma unroll
            for (int i = 0; i < 8; ++i) direct_load_b128_nt(rsrc_b, my_lds + buf * BUF + i * 1024, (w_in >> i) & 1 ? w_off[i] : kOutOfRange, k0);
#pragma unroll
            for (int i = 0; i < A_LOADS; ++i) direct_load_b128(rsrc_a, a_lds + buf * ABUF + (wave + i * NW) * 1024, (a_in >> i) & 1 ? a_off[i] : kOutOfRange, k0);
            return;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) direct_load_b128_nt(rsrc_b, my_lds + buf * BUF + i * 1024, w_off[i], k0);
#pragma unroll
        for (int i = 0; i < A_LOADS; ++i) direct_load_b128(rsrc_a, a_lds + buf * ABUF + (wave + i * NW) * 1024, a_off[i], k0);
    };

    // a lane holds four consecutive weight rows' results; their scales, asked for in front of everything else
    const int col = n_base + lg * 4;
    const float* sb = p.sb + (int64_t)expert * N * p.sb_step;
    float s[4], b[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int c = min(col + q, N - 1);
        s[q] = sb[(int64_t)c * p.sb_step];
        b[q] = load_bias(p.bias, p.bias_type, c);
    }
    float sa[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) sa[mt] = p.sa[(row0 + min(mt * 16 + li, rows_a - 1)) * p.sa_step];

    v4i acc[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) acc[mt] = v4i{0, 0, 0, 0};
    constexpr int kBut = 8 + A_LOADS;  // all but the loads of one piece
    constexpr int kWaitBut = 0x0F70 | (kBut & 15) | ((kBut >> 4) << 14);
    constexpr int kWaitAll = 0x0F70, kWaitLds = 0xC07F;
    const int n_pieces = max(c_end - c_begin, 0);
    const int rot = n_pieces > 0 ? (int)(blockIdx.x % (unsigned)n_pieces) : 0;
    auto piece = [&](int i) { const int c = c_begin + i + rot; return c >= c_end ? c - n_pieces : c; };
    if (0 < n_pieces) issue(piece(0), 0);
    if (1 < n_pieces) issue(piece(1), 1);
    for (int it = 0; it < n_pieces; ++it) {
        const int buf = it & 1;
        // my loads of this piece have landed (those of the next may be in flight) ...
        if (it + 1 >= n_pieces) __builtin_amdgcn_s_waitcnt(kWaitAll);
        else __builtin_amdgcn_s_waitcnt(kWaitBut);
        __builtin_amdgcn_s_barrier();  // ... and so has every other wave's share of the activation piece
        const uint8_t* wb = my_buf + buf * BUF + li * PIECE;
        const uint8_t* ab = sA + buf * ABUF + li * PIECE;
        v8i wf[SPC], af[MT][SPC];
#pragma unroll
        for (int s = 0; s < SPC; ++s) {
            const int j0 = ((s * 8 + lg) ^ li) << 4, j1 = ((s * 8 + 4 + lg) ^ li) << 4;
            wf[s] = join(*reinterpret_cast<const v4i*>(wb + j0), *reinterpret_cast<const v4i*>(wb + j1));
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
                af[mt][s] = join(*reinterpret_cast<const v4i*>(ab + mt * BUF + j0), *reinterpret_cast<const v4i*>(ab + mt * BUF + j1));
        }
        __builtin_amdgcn_s_waitcnt(kWaitLds);
#pragma unroll
        for (int s = 0; s < SPC; ++s) {
            asm volatile("" : "+v"(wf[s]));
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) asm volatile("" : "+v"(af[mt][s]));
        }
        __builtin_amdgcn_s_barrier();  // every wave holds its fragments: this buffer may be refilled
        if (it + 2 < n_pieces) issue(piece(it + 2), buf);
#pragma unroll
        for (int s = 0; s < SPC; ++s) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) acc[mt] = mfma_i8(lo4(wf[s]), lo4(af[mt][s]), acc[mt]);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) acc[mt] = mfma_i8(hi4(wf[s]), hi4(af[mt][s]), acc[mt]);
        }
    }
    // (n_end cuts off those of the four that are not the wave's)
    if (col >= n_end) return;
    const bool vec_ok = p.vec_store != 0 && (R & 3) == 0;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int m = mt * 16 + li;
        if (m >= rows_a) continue;
        if (!RAGGED && p.split_k > 1) {
            int* mine = p.partials + ((int64_t)blockIdx.y * p.M + m) * N + col;
            if (vec_ok) {
                *reinterpret_cast<v4i*>(mine) = acc[mt];
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (col + q < n_end) mine[q] = acc[mt][q];
            }
            continue;
        }
        v4f y;
#pragma unroll
        for (int q = 0; q < 4; ++q) y[q] = finish(acc[mt][q], sa[mt], s[q], b[q]);
        store4(p.C, p.out_type, row0 + m, col, n_end, (int)p.ldc, y, 0.f, vec_ok);
    }
#endif
}

}  // namespace tg
