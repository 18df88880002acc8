// Rows in int8 with a scale each, in front of a product in 8-bit integers:
//   y = x, or silu(gate) * up of a row that holds both halves (fp32, not rounded between)
//   scale = max|y| * fp32(1 / 127) (an all-zero row: 1);  q = round-half-even(y / scale), an IEEE quotient, within +-127
// A row that holds a NaN or an infinity gets the scale NaN and codes of zero, so that it shows in what is
// multiplied with it.  With `place` a row's codes go to several rows: tokens on their way to the experts that each of them was sent to.
//
// Bound by HBM (a row is read once and stays in the registers of the lanes that share it, V vectors of 8 elements each), few rows by latency: 5000 x 14336 f16 42 us (5.1 TB/s),
// 24576 x 1408 activated bf16 31 (5.6), 4096 x 2048 to six places each 17 (4.0).
// Rows longer than the registers of 1024 lanes are read twice.
#include "quant_device.h"

namespace tg {
namespace {

// 8 elements from `at`; where the rows are not aligned to vectors element by element, zeros behind `end`.
template <typename T, bool VEC>
__device__ __forceinline__ v8f_q fetch8(const T* p, int at, int end) {
    if constexpr (VEC) return load8<T>(p + at);
    v8f_q v;
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = at + k < end ? (float)p[at + k] : 0.f;
    return v;
}

__device__ __forceinline__ float silu_mul(float gate, float up) { return gate * __builtin_amdgcn_rcpf(1.0f + __expf(-gate)) * up; }

// Eight elements of the row whose codes are wanted.
template <typename T, bool ACT, bool VEC>
__device__ __forceinline__ v8f_q row8(const T* x, int at, int K) {
    v8f_q v = fetch8<T, VEC>(x, at, K);
    if constexpr (ACT) {
        const v8f_q up = fetch8<T, VEC>(x + K, at, K);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = silu_mul(v[k], up[k]);
    }
    return v;
}

// Magnitudes as bit patterns: their order is that of the numbers, with infinity and NaN above all of them.
__device__ __forceinline__ uint32_t magnitude(v8f_q v) {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) m = max(m, __float_as_uint(v[k]) & 0x7FFFFFFFu);
    return m;
}

__device__ __forceinline__ v2i codes8(v8f_q v, const ScaleDivider& d) {
    // 1.5 * 2^23 added to a number below 2^22 rounds it half to even, and leaves the integer in the low bits
    uint32_t c[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        float t;
        if (d.fast) {  // (|t| < 127.5: the scale is max|y| / 127 to three roundings)
            t = v[k] * d.r;
            t = __builtin_fmaf(-__builtin_fmaf(d.s, t, -v[k]), d.r, t);
            t = __builtin_fmaf(-__builtin_fmaf(d.s, t, -v[k]), d.r, t);
        } else {
            t = __builtin_amdgcn_fmed3f(v[k] / d.s, -127.f, 127.f);
        }
        c[k] = __float_as_uint(t + 0x1.8p23f);
    }
    auto low_bytes = [](uint32_t a, uint32_t b, uint32_t e, uint32_t f) {
        return (int)(__builtin_amdgcn_perm(b, a, 0x0c0c0400u) | __builtin_amdgcn_perm(f, e, 0x04000c0cu));
    };
    return v2i{low_bytes(c[0], c[1], c[2], c[3]), low_bytes(c[4], c[5], c[6], c[7])};
}

template <bool VEC>
__device__ __forceinline__ void put8(int8_t* q, int at, int K, v2i c) {
    if constexpr (VEC) {
        *reinterpret_cast<v2i*>(q + at) = c;
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (at + k < K) q[at + k] = (int8_t)(c[k >> 2] >> (8 * (k & 3)));
    }
}

// TPR lanes share a row (64 or 128: four or two rows per workgroup; else the workgroup has one), V vectors of 8 elements per lane; V = 0: as many
// as it takes, read twice.
template <typename T, bool ACT, bool VEC, bool PLACE, int TPR, int V>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) int8_quant_kernel(const Int8QuantParams p) {
    constexpr int ROWS = TPR < 256 ? 256 / TPR : 1, WAVES = TPR / 64;
    const int tid = (int)threadIdx.x, lane = tid % TPR, K = p.K;
    const int64_t row = (int64_t)blockIdx.x * ROWS + tid / TPR;
    const bool live = row < p.rows;  // the lanes of a row are in or out together, and whole waves at a time
    const T* x = (const T*)p.x + row * K * (ACT ? 2 : 1);
    v8f_q v[V ? V : 1];
    uint32_t top = 0;
    if constexpr (V > 0) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int at = (i * TPR + lane) * 8;
#pragma unroll
            for (int k = 0; k < 8; ++k) v[i][k] = 0.f;
            if (live && at < K) v[i] = row8<T, ACT, VEC>(x, at, K);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) top = max(top, magnitude(v[i]));
    } else if (live) {
        for (int at = lane * 8; at < K; at += TPR * 8) top = max(top, magnitude(row8<T, ACT, VEC>(x, at, K)));
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
    if constexpr (WAVES > 1) {
        __shared__ uint32_t part[ROWS * WAVES];
        if (tid % 64 == 0) part[tid / 64] = top;
        __syncthreads();
        top = 0;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) top = max(top, part[tid / TPR * WAVES + i]);
    }
    if (!live) return;
    const bool number = top < 0x7F800000u;
    const float amax = __uint_as_float(top);
    float scale = amax * (1.0f / 127.0f);
    if (scale == 0.f) scale = 1.f;  // (the smallest subnormal rows with it: their codes are zeros)
    if (!number) scale = __uint_as_float(0x7FC00000u);
    const ScaleDivider div(number ? scale : 1.f);
    auto emit = [&](int at, v8f_q w) {
        const v2i c = number ? codes8(w, div) : v2i{0, 0};
        if constexpr (PLACE) {
            for (int j = 0; j < p.copies; ++j) {
                int64_t to = p.place[row * p.copies + j];
                const bool none = to < 0;
                if (none) to = -1 - to;
                if (to < p.places) put8<VEC>(p.q + to * K, at, K, none ? v2i{0, 0} : c);
            }
        } else {
            put8<VEC>(p.q + row * K, at, K, c);
        }
    };
    if constexpr (V > 0) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int at = (i * TPR + lane) * 8;
            if (at < K) emit(at, v[i]);
        }
    } else {
        for (int at = lane * 8; at < K; at += TPR * 8) emit(at, row8<T, ACT, VEC>(x, at, K));
    }
    if constexpr (PLACE) {
        for (int j = lane; j < p.copies; j += TPR) {
            const int64_t place = p.place[row * p.copies + j], to = place < 0 ? -1 - place : place;
            if (to < p.places) p.scales[to] = place < 0 ? 1.f : scale;
        }
    } else if (lane == 0) {
        p.scales[row] = scale;
    }
}

// (rows from which a wave has one to itself, us with / without: 2048 x 1408 activated 7.6 / 8.5, 24576 x 1408 34.5 / 48, 65536 x 1024 36 / 51)
constexpr int64_t kWaveRows = 2048;
// As many lanes as a row has vectors, one each: a row's chain of load, maximum, exchange, store is shortest.  With many rows, a
// wave for each of up to 256 vectors: no lanes without a vector but in the last sixty-four, and nothing is exchanged through LDS.
int lanes_of(const Int8QuantParams& p) {
    const int vectors = (p.K + 7) / 8;
    if (p.rows >= kWaveRows && vectors <= 256) return 64;
    return vectors <= 64 ? 64 : vectors <= 128 ? 128 : vectors <= 256 ? 256 : vectors <= 512 ? 512 : 1024;
}
int64_t blocks_of(const Int8QuantParams& p, int lanes) {
    const int rows = lanes < 256 ? 256 / lanes : 1;
    return (p.rows + rows - 1) / rows;
}

template <typename T, bool ACT, bool VEC, bool PLACE>
hipError_t launch(const Int8QuantParams& p, hipStream_t s) {
    const int vectors = (p.K + 7) / 8, lanes = lanes_of(p);
    const dim3 grid((unsigned)blocks_of(p, lanes)), block(lanes < 256 ? 256 : lanes);
#define TG_QUANT(TPR, V)                                                                             \
    if (lanes == TPR && (V == 0 || vectors <= TPR * V)) {                                            \
        hipLaunchKernelGGL((int8_quant_kernel<T, ACT, VEC, PLACE, TPR, V>), grid, block, 0, s, p);   \
        return hipGetLastError();                                                                    \
    }
    TG_QUANT(64, 1)
    TG_QUANT(64, 2)
    TG_QUANT(64, 3)
    TG_QUANT(64, 4)
    TG_QUANT(128, 1)
    TG_QUANT(256, 1)
    TG_QUANT(512, 1)
    TG_QUANT(1024, 1)
    TG_QUANT(1024, 2)
    TG_QUANT(1024, 4)
    TG_QUANT(1024, 0)
#undef TG_QUANT
    return hipErrorInvalidValue;
}

template <typename T>
hipError_t launch_type(const Int8QuantParams& p, hipStream_t s) {
    // rows of x and of q start on 16- and 8-byte boundaries
    const bool vec = p.K % 8 == 0 && reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && reinterpret_cast<uintptr_t>(p.q) % 8 == 0;
    if (p.place) return vec ? launch<T, false, true, true>(p, s) : launch<T, false, false, true>(p, s);
    if (p.silu_mul) return vec ? launch<T, true, true, false>(p, s) : launch<T, true, false, false>(p, s);
    return vec ? launch<T, false, true, false>(p, s) : launch<T, false, false, false>(p, s);
}

}  // namespace

int64_t int8_quant_threads(const Int8QuantParams& p) {
    const int lanes = lanes_of(p);
    return blocks_of(p, lanes) * (lanes < 256 ? 256 : lanes);
}

hipError_t run_int8_quant(const Int8QuantParams& p, int x_type, hipStream_t s) {
    if (p.rows <= 0) return hipSuccess;
    if (x_type == OUT_F32) return launch_type<float>(p, s);
    if (x_type == OUT_BF16) return launch_type<__bf16>(p, s);
    if (x_type == OUT_F16) return launch_type<_Float16>(p, s);
    return hipErrorInvalidValue;
}

}  // namespace tg
