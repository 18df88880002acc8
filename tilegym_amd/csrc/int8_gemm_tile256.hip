// Instantiation of the 256 x 256 int8 tiles.
#include "int8_gemm_tile256.h"

namespace tg {

hipError_t run_int8_tile256(const Int8GemmParams& p, hipStream_t s) {
    if (p.K % kKBlock != 0 || p.K < 2 * kKBlock || (int64_t)p.M * p.K >= ((int64_t)1 << 31) || (int64_t)p.N * p.K >= ((int64_t)1 << 31)) return hipErrorInvalidValue;
    const int64_t tiles = (((int64_t)p.M + 255) / 256) * ((p.N + 255) / 256);
    const int units = compute_units();
    const dim3 grid((unsigned)(tiles < units ? tiles : units)), block(256);
#define TG_CASE(OT, BIAS)                                                                            \
    if (p.out_type == OT && bias_kind(p) == BIAS) {                                                  \
        hipLaunchKernelGGL((int8_gemm_tile256_kernel<OT, BIAS>), grid, block, 0, s, p);              \
        return hipGetLastError();                                                                    \
    }
    TG_CASE(OUT_BF16, BIAS_NONE) TG_CASE(OUT_BF16, BIAS_F32) TG_CASE(OUT_BF16, BIAS_16)
    TG_CASE(OUT_F16, BIAS_NONE) TG_CASE(OUT_F16, BIAS_F32) TG_CASE(OUT_F16, BIAS_16)
    TG_CASE(OUT_F32, BIAS_NONE) TG_CASE(OUT_F32, BIAS_F32) TG_CASE(OUT_F32, BIAS_16)
#undef TG_CASE
    return hipErrorInvalidValue;
}

}  // namespace tg
