// Root-mean-square norm with the residual's addition and an e4m3 output, in front of an FP8 projection:
//   s = x + r                       fp32; written back rounded to x's type where the caller asks for it
//   y = s * rsqrt(mean(s^2) + eps) * w
//   q = rne_e4m3(clamp(y / scale, -448, 448))
//   scale = amax(|y|) / 448 over groups of 16, 32, 64 or 128 consecutive elements (all-zero group -> 1), the rule of act_quant,
//           or one given scale for the whole tensor
// The norm is taken of the fp32 sum and y goes to e4m3 without a 16-bit rounding between: one rounding in place of three
// launches' three.  Both divisions are IEEE quotients, so codes and scales are the bits of act_quant on the fp32 norm (with a product by the reciprocal in
// their place one code in a million is another: 777 x 5120 8.15 us, 8.4 with quotients; 8192 x 4096 43.1 and 43.3).
//
// Bound by HBM (at most 3 x 16 bits + 1 byte per element), few rows by latency: a row is read once and stays in the registers of the lanes that
// share it, V vectors of 8 elements each; the two reductions are the sum of squares over the row and the maximum over the 2 to
// 16 neighbouring lanes of a group.
#include "quant_device.h"

namespace tg {
namespace {

template <typename T>
struct Vec8 { typedef T type __attribute__((ext_vector_type(8))); };

template <typename T>
__device__ __forceinline__ void store8(T* p, v8f_q v) {
    *reinterpret_cast<typename Vec8<T>::type*>(p) = __builtin_convertvector(v, typename Vec8<T>::type);
}
template <>
__device__ __forceinline__ void store8<float>(float* p, v8f_q v) {
    reinterpret_cast<v4f*>(p)[0] = __builtin_shufflevector(v, v, 0, 1, 2, 3);
    reinterpret_cast<v4f*>(p)[1] = __builtin_shufflevector(v, v, 4, 5, 6, 7);
}

// ScaleDivider's quotient, with residuals s t - a that are subtracted: a zero keeps its sign by itself.
__device__ __forceinline__ float quotient(float a, const ScaleDivider& d) {
    float t = a * d.r;
    t = __builtin_fmaf(-__builtin_fmaf(d.s, t, -a), d.r, t);
    return __builtin_fmaf(-__builtin_fmaf(d.s, t, -a), d.r, t);
}

// TPR lanes share a row (64 or 128: four or two rows per workgroup; else the workgroup has one), V vectors of 8 elements per lane.
// x, r and their outputs may be the same memory (element by element): no __restrict__ on them.
template <typename T, typename W, int TPR, int V>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) rms_norm_quant_kernel(const NormQuantParams p) {
    constexpr int ROWS = TPR < 256 ? 256 / TPR : 1, WAVES = TPR / 64;
    const int tid = (int)threadIdx.x, lane = tid % TPR;
    const int64_t row = (int64_t)blockIdx.x * ROWS + tid / TPR;
    const bool live = row < p.rows;  // the lanes of a row are in or out together, and whole waves at a time
    const int vectors = p.hidden / 8;
    const T* x = (const T*)p.x + row * p.hidden;
    const T* r = (const T*)p.residual + row * p.hidden;
    constexpr bool EARLY = V <= 2;  // the weights' loads in front of the reduction; with more vectors they would cost registers
    v8f_q v[V], w[EARLY ? V : 1];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int at = i * TPR + lane;
#pragma unroll
        for (int k = 0; k < 8; ++k) v[i][k] = 0.f;
        if (live && at < vectors) {
            v[i] = load8<T>(x + at * 8);
            if constexpr (EARLY) w[i] = load8<W>((const W*)p.weight + at * 8);
        }
    }
    if (p.residual) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int at = i * TPR + lane;
            if (live && at < vectors) v[i] += load8<T>(r + at * 8);
        }
    }
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) sum = __builtin_fmaf(v[i][k], v[i][k], sum);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
    if constexpr (WAVES > 1) {
        __shared__ float part[ROWS * WAVES];
        if (tid % 64 == 0) part[tid / 64] = sum;
        __syncthreads();
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) sum += part[tid / TPR * WAVES + i];
    }
    if (!live) return;
    const float norm = 1.0f / sqrtf(sum / (float)p.hidden + p.eps);
    float given = 1.f;
    if (p.scale) given = *p.scale;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int at = i * TPR + lane;
        if (at < vectors) {  // (a group's lanes together: hidden is a multiple of the group)
            if (p.residual_out) store8<T>((T*)p.residual_out + row * p.hidden + at * 8, v[i]);
            v8f_q y;
            const v8f_q wi = EARLY ? w[EARLY ? i : 0] : load8<W>((const W*)p.weight + at * 8);
#pragma unroll
            for (int k = 0; k < 8; ++k) y[k] = v[i][k] * norm * wi[k];
            if (p.norm_out) store8<T>((T*)p.norm_out + row * p.hidden + at * 8, y);
            float s = given;
            if (!p.scale) {
                float amax = 0.f;
#pragma unroll
                for (int k = 0; k < 8; ++k) amax = fmaxf(amax, fabsf(y[k]));
                amax = dpp_max<0xB1>(amax);
                if (p.lanes_per_group >= 4) amax = dpp_max<0x4E>(amax);
                if (p.lanes_per_group >= 8) amax = dpp_max<0x141>(amax);
                if (p.lanes_per_group >= 16) amax = dpp_max<0x140>(amax);
                s = amax == 0.f ? 1.0f : amax / 448.0f;
                if ((at & (p.lanes_per_group - 1)) == 0) p.scales[row * (vectors >> p.group_shift) + (at >> p.group_shift)] = s;
            }
            v8f_q c;
            const ScaleDivider div(s);
            if (div.fast) {
                if (p.scale) {  // infinite and very large y are cut where the code saturates anyway, before their residuals are no numbers
#pragma unroll
                    for (int k = 0; k < 8; ++k) y[k] = __builtin_amdgcn_fmed3f(y[k], -512.0f * s, 512.0f * s);
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) c[k] = quotient(y[k], div);
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) c[k] = y[k] / s;
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) c[k] = __builtin_amdgcn_fmed3f(c[k], -448.0f, 448.0f);
            int packed[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                int b = 0;
                b = __builtin_amdgcn_cvt_pk_fp8_f32(c[4 * h], c[4 * h + 1], b, false);
                b = __builtin_amdgcn_cvt_pk_fp8_f32(c[4 * h + 2], c[4 * h + 3], b, true);
                packed[h] = b;
            }
            *reinterpret_cast<v2i*>(p.q + row * p.hidden + at * 8) = v2i{packed[0], packed[1]};
        }
        if constexpr (V > 2) __builtin_amdgcn_sched_barrier(0);  // one vector's temporaries at a time
    }
}

// As many lanes as a row has vectors, one each: a row's chain of load, sum, exchange, store is shortest, and few registers let many rows share
// a compute unit (kernel and launch, bf16 with residual, one vector per lane against up to four on 256 lanes: 1 x 4096 3.5 / 4.3 us,
// 777 x 5120 9.7 / 13.5, 4096 x 8192 49.3 / 85.0, 1000 x 16384 with two on 1024 24.8 / 39.8).  Rows of 4097 to 8192 elements leave lanes of 1024 idle:
// with enough rows to fill the chip two vectors on 512 are ahead (777 x 5120 9.0 / 9.7 us, 2000 x 8192 24.2 / 25.7; one row of 8192 4.1 / 3.9).
// 8192 x 4096 with one given scale, call after call: 43.3 us, 5.4 TB/s, as part of the 235 MB stays in the caches (a copy: 5.2 TB/s, 45 us).
int lanes_of(const NormQuantParams& p) {
    const int vectors = p.hidden / 8;
    if (vectors <= 512) return vectors <= 64 ? 64 : vectors <= 128 ? 128 : vectors <= 256 ? 256 : 512;
    return vectors > 2048 || (vectors <= 1024 && p.rows >= 512) ? 512 : 1024;
}
int64_t blocks_of(const NormQuantParams& p, int lanes) {
    const int rows = lanes < 256 ? 256 / lanes : 1;
    return (p.rows + rows - 1) / rows;
}

template <typename T, typename W>
hipError_t launch(const NormQuantParams& p, hipStream_t s) {
    const int vectors = p.hidden / 8, lanes = lanes_of(p);
    const dim3 grid((unsigned)blocks_of(p, lanes)), block(lanes < 256 ? 256 : lanes);
#define TG_NORM(TPR, V)                                                                            \
    if (lanes == TPR && vectors <= TPR * V) {                                                      \
        hipLaunchKernelGGL((rms_norm_quant_kernel<T, W, TPR, V>), grid, block, 0, s, p);           \
        return hipGetLastError();                                                                  \
    }
    TG_NORM(64, 1)
    TG_NORM(128, 1)
    TG_NORM(256, 1)
    TG_NORM(512, 1)
    TG_NORM(512, 2)
    TG_NORM(1024, 1)
    TG_NORM(1024, 2)
    TG_NORM(512, 8)
#undef TG_NORM
    return hipErrorInvalidValue;
}

}  // namespace

int64_t rms_norm_quant_threads(const NormQuantParams& p) {
    const int lanes = lanes_of(p);
    return blocks_of(p, lanes) * (lanes < 256 ? 256 : lanes);
}

hipError_t run_rms_norm_quant(const NormQuantParams& p, int x_type, bool weight_f32, hipStream_t s) {
    if (p.rows <= 0) return hipSuccess;
    if (x_type == OUT_F32) return launch<float, float>(p, s);
    if (x_type == OUT_BF16) return weight_f32 ? launch<__bf16, float>(p, s) : launch<__bf16, __bf16>(p, s);
    if (x_type == OUT_F16) return weight_f32 ? launch<_Float16, float>(p, s) : launch<_Float16, _Float16>(p, s);
    return hipErrorInvalidValue;
}

}  // namespace tg
