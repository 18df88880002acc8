// Instantiation of the 256 x 256 int8 tiles.
#include "int8_gemm_tile256.h"

namespace tg {

hipError_t run_int8_tile256(const Int8GemmParams& p, hipStream_t s) {
    if (p.K % kKBlock != 0 || p.K < 2 * kKBlock || (int64_t)p.M * p.K >= ((int64_t)1 << 31) || (int64_t)p.N * p.K >= ((int64_t)1 << 31)) return hipErrorInvalidValue;
    const int64_t row_tiles = p.m_indptr ? most_row_tiles(p.M, p.E, 256) : ((int64_t)p.M + 255) / 256, tiles = row_tiles * ((p.N + 255) / 256);
    if (tiles > INT32_MAX / 2) return hipErrorInvalidValue;
    const int64_t units = compute_units();
    const dim3 grid((unsigned)(p.m_indptr ? walking_grid(tiles, units) : tiles < units ? tiles : units)), block(256);
    if (p.m_indptr && p.bias) return hipErrorInvalidValue;
#define TG_LAUNCH(OT, BIAS, RAGGED)                                                                  \
    {                                                                                                \
        hipLaunchKernelGGL((int8_gemm_tile256_kernel<OT, BIAS, RAGGED>), grid, block, 0, s, p);      \
        return hipGetLastError();                                                                    \
    }
    if (p.m_indptr) {
        if (p.out_type == OUT_BF16) TG_LAUNCH(OUT_BF16, BIAS_NONE, true)
        if (p.out_type == OUT_F16) TG_LAUNCH(OUT_F16, BIAS_NONE, true)
        if (p.out_type == OUT_F32) TG_LAUNCH(OUT_F32, BIAS_NONE, true)
        return hipErrorInvalidValue;
    }
#define TG_CASE(OT, BIAS) \
    if (p.out_type == OT && bias_kind(p) == BIAS) TG_LAUNCH(OT, BIAS, false)
    TG_CASE(OUT_BF16, BIAS_NONE) TG_CASE(OUT_BF16, BIAS_F32) TG_CASE(OUT_BF16, BIAS_16)
    TG_CASE(OUT_F16, BIAS_NONE) TG_CASE(OUT_F16, BIAS_F32) TG_CASE(OUT_F16, BIAS_16)
    TG_CASE(OUT_F32, BIAS_NONE) TG_CASE(OUT_F32, BIAS_F32) TG_CASE(OUT_F32, BIAS_16)
#undef TG_CASE
#undef TG_LAUNCH
    return hipErrorInvalidValue;
}

}  // namespace tg
