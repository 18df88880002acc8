// Products in 8-bit integers for operands that the kernels with direct loads do not take: rows whose length or address is no multiple of
// 16 bytes.
//
// A workgroup of four waves makes 64 x 64 outputs.  Both operands go through registers to LDS, 64 bytes of K at a time: a thread fetches
// 16 bytes of one row at any address (the tail of a row byte by byte, zeros beyond it), one step ahead of the MFMAs.  Rows of LDS are 80
// bytes apart, so that the sixteen rows a fragment read touches start in different banks.  Bound by the latency of that one
// step (0.6 us), so K is split where tiles are few: 512 x 1001 x 1003 takes 12.7 us, 4096 x 4099 x 4095 306 (449 TOP/s); 8 x 4096 x 4096 from an odd address, for which
// the Python calls bring no scratch memory, 24 where an aligned call takes 6.6.
#include "int8_device.h"

namespace tg {
namespace {

[[maybe_unused]] constexpr int kPitch = 80;

// 16 bytes at p, which has no alignment; `have` of them belong to the row.
[[maybe_unused]] __device__ __forceinline__ v4i fetch16(const int8_t* p, int64_t have) {
    v4i v = v4i{0, 0, 0, 0};
    if (have >= 16) {
        __builtin_memcpy(&v, p, 16);
    } else if (have > 0) {
        int8_t b[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) b[i] = i < have ? p[i] : (int8_t)0;
        __builtin_memcpy(&v, b, 16);
    }
    return v;
}

template <bool RAGGED>
__global__ void __launch_bounds__(256) int8_gemm_simple_kernel(const Int8GemmParams p) {
#if defined(__HIP_DEVICE_COMPILE__)
    __shared__ __align__(16) int8_t sA[2][64 * kPitch], sB[2][64 * kPitch];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int tiles_n = (p.N + 63) / 64;
    int expert = 0, n0 = blockIdx.x % tiles_n * 64, rows_valid;
    int64_t m0 = (int64_t)(blockIdx.x / tiles_n) * 64;
    if constexpr (RAGGED) {
        int tile_n;
        if (!ragged_tile<64>(p, (int)blockIdx.x, tiles_n, lane, expert, m0, rows_valid, tile_n)) return;
        n0 = tile_n * 64;
    } else {
        rows_valid = (int)min((int64_t)64, p.M - m0);
    }
    const int64_t m_end = m0 + rows_valid;
    const int row = tid >> 2, at = (tid & 3) * 16;  // what this thread fetches
    const bool has_a = m0 + row < m_end, has_b = n0 + row < p.N;
    const int8_t* a = p.A + (m0 + row) * (int64_t)p.K + at;
    const int8_t* b = p.B + ((int64_t)expert * p.N + n0 + row) * (int64_t)p.K + at;
    int steps = (p.K + 63) / 64, s0 = 0;
    if (!RAGGED && p.split_k > 1) {
        s0 = 2 * (int)blockIdx.y * p.ksteps_per_split;
        steps = min(s0 + 2 * p.ksteps_per_split, steps);
    }
    auto left = [&](bool has, int step) { return has ? (int64_t)p.K - (int64_t)step * 64 - at : (int64_t)0; };
    v4i ra = fetch16(a + (int64_t)s0 * 64, left(has_a, s0)), rb = fetch16(b + (int64_t)s0 * 64, left(has_b, s0));
    const int wm = wave & 1, wn = wave >> 1, li = lane & 15, lg = lane >> 4;
    v4i acc[2][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i >> 1][i & 1] = v4i{0, 0, 0, 0};
    for (int s = s0; s < steps; ++s) {
        *reinterpret_cast<v4i*>(&sA[s & 1][row * kPitch + at]) = ra;
        *reinterpret_cast<v4i*>(&sB[s & 1][row * kPitch + at]) = rb;
        __syncthreads();  // (the other buffer's readers have passed the barrier of the step before)
        if (s + 1 < steps) {
            ra = fetch16(a + (int64_t)(s + 1) * 64, left(has_a, s + 1));
            rb = fetch16(b + (int64_t)(s + 1) * 64, left(has_b, s + 1));
        }
        v4i fa[2], fb[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            fa[t] = *reinterpret_cast<const v4i*>(&sA[s & 1][(wm * 32 + t * 16 + li) * kPitch + lg * 16]);
            fb[t] = *reinterpret_cast<const v4i*>(&sB[s & 1][(wn * 32 + t * 16 + li) * kPitch + lg * 16]);
        }
#pragma unroll
        for (int tn = 0; tn < 2; ++tn)
#pragma unroll
            for (int tm = 0; tm < 2; ++tm) acc[tn][tm] = mfma_i8(fb[tn], fa[tm], acc[tn][tm]);
    }
#pragma unroll
    for (int tm = 0; tm < 2; ++tm) {
        const int64_t m = m0 + wm * 32 + tm * 16 + li;
        if (m >= m_end) continue;
        if (!RAGGED && p.split_k > 1) {
            int* const mine = p.partials + ((int64_t)blockIdx.y * p.M + m) * p.N;
#pragma unroll
            for (int tn = 0; tn < 2; ++tn)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int n = n0 + wn * 32 + tn * 16 + lg * 4 + r;
                    if (n < p.N) mine[n] = acc[tn][tm][r];
                }
            continue;
        }
        const float sa = p.sa[m * p.sa_step];
#pragma unroll
        for (int tn = 0; tn < 2; ++tn)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int n = n0 + wn * 32 + tn * 16 + lg * 4 + r;
                if (n >= p.N) continue;
                put1(p, m * p.ldc + n, finish(acc[tn][tm][r], sa, p.sb[((int64_t)expert * p.N + n) * p.sb_step], load_bias(p.bias, p.bias_type, n)));
            }
    }
#endif
}

}  // namespace

int64_t int8_simple_threads(const Int8GemmParams& p) {
    const int64_t row_tiles = p.m_indptr ? most_row_tiles(p.M, p.E, 64) : ((int64_t)p.M + 63) / 64;
    return row_tiles * (((int64_t)p.N + 63) / 64) * 256 * p.split_k;
}

hipError_t run_int8_simple(const Int8GemmParams& p, hipStream_t s) {
    const dim3 grid((unsigned)(int8_simple_threads(p) / 256 / p.split_k), p.split_k);
    if (p.m_indptr) hipLaunchKernelGGL(int8_gemm_simple_kernel<true>, grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL(int8_gemm_simple_kernel<false>, grid, dim3(256), 0, s, p);
    return hipGetLastError();
}

}  // namespace tg
