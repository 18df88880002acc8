// Instantiations of the int8 ring tiles, and the sum of a split K.
#include "int8_gemm_ring.h"

namespace tg {
namespace {

// One thread adds the partial sums of four neighbouring outputs and finishes them.
__global__ void __launch_bounds__(256) int8_splitk_reduce_kernel(const Int8GemmParams p) {
    const int64_t quads = ((int64_t)p.N + 3) / 4, idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (idx >= quads * p.M) return;
    const int m = (int)(idx / quads), col = (int)(idx % quads) * 4;
    const int64_t MN = (int64_t)p.M * p.N, at = (int64_t)m * p.N + col;
    v4i sum = v4i{0, 0, 0, 0};
    if (p.N % 4 == 0) {
        for (int z = 0; z < p.split_k; z += 4) {  // four loads in flight
            v4i t[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) t[i] = z + i < p.split_k ? __builtin_nontemporal_load(reinterpret_cast<const v4i*>(p.partials + (z + i) * MN + at)) : v4i{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 4; ++i) sum += t[i];
        }
    } else {
        for (int z = 0; z < p.split_k; ++z)
            for (int q = 0; q < 4 && col + q < p.N; ++q) sum[q] += p.partials[z * MN + at + q];
    }
    const float sa = p.sa[(int64_t)m * p.sa_step];
    v4f y;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int c = min(col + q, p.N - 1);
        y[q] = finish(sum[q], sa, p.sb[(int64_t)c * p.sb_step], load_bias(p.bias, p.bias_type, c));
    }
    store4(p.C, p.out_type, m, col, p.N, (int)p.ldc, y, 0.f, p.vec_store != 0);
}

}  // namespace

// Stages: as many as 160 KiB hold, up to twelve.
#define TG_RING_TILES(X) \
    X(64, 32, 12) X(32, 64, 12) X(64, 64, 9) X(64, 128, 5) X(96, 128, 4) X(128, 128, 4) X(160, 128, 4) X(160, 192, 3) X(192, 192, 3) X(256, 128, 3)

bool int8_ring_exists(int bm, int bn) {
#define TG_IS(BM, BN, STAGES) || (bm == BM && bn == BN)
    return false TG_RING_TILES(TG_IS);
#undef TG_IS
}

hipError_t run_int8_ring(int bm, int bn, const Int8GemmParams& p, hipStream_t s) {
    if (p.K % 16 != 0) return hipErrorInvalidValue;
#define TG_CASE(BM, BN, STAGES) \
    if (bm == BM && bn == BN) return launch_int8_ring<BM, BN, STAGES>(p, s);
    TG_RING_TILES(TG_CASE)
#undef TG_CASE
    return hipErrorInvalidConfiguration;
}

hipError_t run_int8_splitk_reduce(const Int8GemmParams& p, hipStream_t s) {
    const int64_t threads = ((int64_t)p.N + 3) / 4 * p.M;
    if (threads > kMostThreads) return hipErrorInvalidValue;
    hipLaunchKernelGGL(int8_splitk_reduce_kernel, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, s, p);
    return hipGetLastError();
}

}  // namespace tg
