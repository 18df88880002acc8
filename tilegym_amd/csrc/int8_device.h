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

// One output from its integer sum.  Three roundings at most beside the store's: the sum's conversion (exact to 2^24), the product with the
// token's scale, and one multiply-add with the channel's scale and the bias.
__device__ __forceinline__ float finish(int sum, float sa, float sb, float bias) { return __builtin_fmaf((float)sum * sa, sb, bias); }

template <typename T>
__device__ __forceinline__ float load_any(const void* p, int64_t i) { return (float)((const T*)p)[i]; }
__device__ __forceinline__ float load_bias(const void* p, int type, int64_t i) {
    if (!p) return 0.f;
    return type == OUT_F32 ? load_any<float>(p, i) : type == OUT_BF16 ? load_any<__bf16>(p, i) : load_any<_Float16>(p, i);
}

}  // namespace tg
