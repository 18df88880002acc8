// Instantiations of the int8 streaming kernel.
#include "int8_gemm_stream.h"

namespace tg {

hipError_t run_int8_stream(const Int8GemmParams& p, hipStream_t s) {
    if (p.K % 16 != 0 || p.wave_rows < 1 || p.wave_rows > 16 || (p.split_k > 1 && (p.m_indptr || p.ksteps_per_split % 4 != 0))) return hipErrorInvalidValue;
    const int64_t gx = ((int64_t)p.N + 4 * p.wave_rows - 1) / (4 * p.wave_rows);
    if (p.m_indptr) {
        // the experts' rows past their first 16: (rows - 1) / 16 passes each, no more than M / 16 in all
        const int64_t gy = (int64_t)p.E + p.M / 16;
        if (gy > 65535 || gx * gy * 256 > kMostThreads) return hipErrorInvalidValue;
        hipLaunchKernelGGL((int8_gemm_stream_kernel<1, true>), dim3((unsigned)gx, (unsigned)gy), dim3(256), 0, s, p);
    } else {
        if (p.M > 32 || p.split_k > 65535) return hipErrorInvalidValue;
        if (p.M <= 16) hipLaunchKernelGGL((int8_gemm_stream_kernel<1, false>), dim3((unsigned)gx, p.split_k), dim3(256), 0, s, p);
        else hipLaunchKernelGGL((int8_gemm_stream_kernel<2, false>), dim3((unsigned)gx, p.split_k), dim3(256), 0, s, p);
    }
    return hipGetLastError();
}

}  // namespace tg
