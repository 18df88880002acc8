// Tokens sorted by expert, carried there and back with the router's weights, and the gradients of both ways.
//
// sort: a stable counting sort of the (token, slot) pairs by expert.  Pairs whose expert is not here (an id outside [0, E)) are sorted behind the
// last expert: every pair has a row, and every row a pair.  Few pairs: every workgroup counts all ids in LDS (those in front of its slice, those
// behind) and ranks its own slice in order: one launch.  Many: a first launch counts each slice, and a workgroup of the second adds the
// slices' counts up.  No order that atomics could change.
//
// permute, unpermute and their gradients go by tokens, not by rows: a token's element is read once and written to its top_k rows, or
// gathered from them, summed in fp32 in the order of the slots and rounded once.  No atomics.  Bound by HBM (8192 tokens x 8 of 2048 bf16: permute 5.3,
// unpermute 4.3, the gradient 4.4 TB/s; 3001 x 8 of 4096 fp32: 4.7, 4.5, 4.2).
#include "quant_device.h"

namespace tg {
namespace {

constexpr int kSortWaves = 16;

// Lanes that hold the same key (keys below 1024), as a mask.
__device__ __forceinline__ unsigned long long same_key(int key, bool in) {
    unsigned long long m = __ballot(in);
#pragma unroll
    for (int b = 0; b < 10; ++b) {
        const bool set = (key >> b) & 1;
        const unsigned long long with = __ballot(set);
        m &= set ? with : ~with;
    }
    return m;
}

template <typename IdT>
__device__ __forceinline__ int expert_of(IdT id, int E) { return id >= 0 && id < E ? (int)id : E; }

// counts[blockIdx][e]: the pairs of expert e in this workgroup's slice.
template <typename IdT>
__global__ void __launch_bounds__(64 * kSortWaves) moe_count_kernel(const IdT* __restrict__ ids, int n, int E, int per_wave, int* __restrict__ counts) {
    extern __shared__ int lds[];
    const int B = E + 1, tid = threadIdx.x;
    constexpr int NT = 64 * kSortWaves;
    for (int i = tid; i < B; i += NT) lds[i] = 0;
    __syncthreads();
    const int64_t lo = (int64_t)blockIdx.x * kSortWaves * per_wave, hi = min(lo + (int64_t)kSortWaves * per_wave, (int64_t)n);
    for (int64_t i = lo + tid; i < hi; i += NT) atomicAdd(&lds[expert_of(ids[i], E)], 1);
    __syncthreads();
    for (int i = tid; i < B; i += NT) counts[(int64_t)blockIdx.x * B + i] = lds[i];
}

template <typename IdT, bool COUNTED>
__global__ void __launch_bounds__(64 * kSortWaves) moe_sort_kernel(const IdT* __restrict__ ids, int n, int E, int per_wave, const int* __restrict__ counts,
                                                                   int* __restrict__ indptr, int* __restrict__ rows, int* __restrict__ slots) {
    extern __shared__ int lds[];
    const int B = E + 1;                   // experts, and the pairs without one
    int* const mine = lds;                 // [kSortWaves][B]: counts of this workgroup's waves, then their next rows
    int* const before = mine + kSortWaves * B;  // [B]: pairs in front of this workgroup's slice
    int* const behind = before + B;        // [B]
    int* const waves = behind + B;         // [kSortWaves]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    constexpr int NT = 64 * kSortWaves;
    for (int i = tid; i < (kSortWaves + 2) * B; i += NT) lds[i] = 0;
    __syncthreads();
    const int64_t lo = (int64_t)blockIdx.x * kSortWaves * per_wave, hi = min(lo + (int64_t)kSortWaves * per_wave, (int64_t)n);
    auto key_of = [&](int64_t i) { return expert_of(ids[i], E); };
    if constexpr (COUNTED) {
        // the slices' counts, several slices at a time; then this workgroup's own, by wave
        const int at_once = NT / B, slice0 = tid / B, e = tid - slice0 * B;
        if (slice0 < at_once) {
            int front = 0, back = 0;
#pragma unroll 8
            for (int g = slice0; g < (int)gridDim.x; g += at_once) {
                const int c = counts[(int64_t)g * B + e];
                front += g < (int)blockIdx.x ? c : 0;
                back += g > (int)blockIdx.x ? c : 0;
            }
            if (front) atomicAdd(&before[e], front);
            if (back) atomicAdd(&behind[e], back);
        }
        const int64_t first = lo + (int64_t)wave * per_wave, last = min(first + per_wave, (int64_t)n);
        for (int64_t i = first + lane; i < last; i += 64) atomicAdd(&mine[wave * B + key_of(i)], 1);
    } else {
        for (int64_t i = tid; i < n; i += NT) {
            const int key = key_of(i);
            if (i < lo) atomicAdd(&before[key], 1);
            else if (i >= hi) atomicAdd(&behind[key], 1);
            else atomicAdd(&mine[(int)(i - lo) / per_wave * B + key], 1);
        }
    }
    __syncthreads();
    // thread e: expert e's pairs, and the rows in front of them
    int total = 0;
    if (tid < B) {
        total = before[tid] + behind[tid];
        for (int w = 0; w < kSortWaves; ++w) total += mine[w * B + tid];
    }
    int upto = total;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int t = __shfl_up(upto, d);
        if (lane >= d) upto += t;
    }
    if (lane == 63) waves[wave] = upto;
    __syncthreads();
    for (int w = 0; w < wave; ++w) upto += waves[w];
    if (tid < B) {
        const int first = upto - total;
        if (blockIdx.x == 0) indptr[tid] = first;
        int next = first + before[tid];
        for (int w = 0; w < kSortWaves; ++w) {
            const int c = mine[w * B + tid];
            mine[w * B + tid] = next;
            next += c;
        }
    }
    __syncthreads();
    volatile int* const cursor = mine + wave * B;  // (written by one lane, read by others of its wave)
    const int64_t first = lo + (int64_t)wave * per_wave, last = min(first + per_wave, (int64_t)n);
    for (int64_t i0 = first; i0 < last; i0 += 64) {
        const int64_t i = i0 + lane;
        const bool in = i < last;
        const int key = in ? key_of(i) : 0;
        const unsigned long long same = same_key(key, in);
        const int rank = __popcll(same & ((1ull << lane) - 1));
        int row = 0;
        if (in) {
            row = cursor[key] + rank;
            rows[i] = key < E ? row : -1 - row;
            slots[row] = (int)i;
        }
        __builtin_amdgcn_wave_barrier();
        if (in && rank == 0) cursor[key] = row + __popcll(same);  // (LDS serves a wave's accesses in their order)
        __builtin_amdgcn_wave_barrier();
    }
}

// ---------------------------------------------------------------------------- there and back
template <typename T, bool VEC>
__device__ __forceinline__ v8f_q get8(const T* p, int at, int H) {
    if constexpr (VEC) return load8<T>(p + at);
    v8f_q v;
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = at + k < H ? (float)p[at + k] : 0.f;
    return v;
}
template <typename T, bool VEC>
__device__ __forceinline__ void set8(T* p, int at, int H, v8f_q v) {
    if constexpr (VEC) {
        if constexpr (sizeof(T) == 4) {
            reinterpret_cast<v4f*>(p + at)[0] = __builtin_shufflevector(v, v, 0, 1, 2, 3);
            reinterpret_cast<v4f*>(p + at)[1] = __builtin_shufflevector(v, v, 4, 5, 6, 7);
        } else {
            typedef T t8 __attribute__((ext_vector_type(8)));
            *reinterpret_cast<t8*>(p + at) = __builtin_convertvector(v, t8);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (at + k < H) p[at + k] = (T)v[k];
    }
}

__device__ __forceinline__ float weight_of(const void* w, int type, int64_t i) {
    return !w ? 1.f : type == OUT_F32 ? ((const float*)w)[i] : type == OUT_BF16 ? (float)((const __bf16*)w)[i] : (float)((const _Float16*)w)[i];
}

constexpr int kRouteLanes = 256;
constexpr int64_t kRoutePairs = 8192;
constexpr int64_t kRouteParts = 65535;  // workgroups up to which a row is shared

// rows[place] = x[token] for each of a token's places; zeros where it has no expert.  Rows are copied in pieces of 16 bytes, element by element where
// they are not aligned to them.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kRouteLanes) moe_permute_kernel(const MoeRouteParams p) {
    constexpr int N = 16 / sizeof(T);
    typedef T piece __attribute__((ext_vector_type(16 / sizeof(T))));
    const int64_t token = blockIdx.x, places = p.tokens * p.top_k;
    const T* x = (const T*)p.x + token * p.H;
    const int* rows = p.rows + token * p.top_k;
    const int step = VEC ? N : 1, lanes = (int)blockDim.x;
    for (int at = ((int)blockIdx.y * lanes + (int)threadIdx.x) * step; at < p.H; at += (int)gridDim.y * lanes * step) {
        piece v, zero;
#pragma unroll
        for (int k = 0; k < N; ++k) zero[k] = (T)0.f;
        if constexpr (VEC) v = *reinterpret_cast<const piece*>(x + at);
        else v[0] = x[at];
        for (int j = 0; j < p.top_k; ++j) {
            const int r = rows[j];
            const int64_t to = r < 0 ? -1 - (int64_t)r : r;
            if (to >= places) continue;
            T* const y = (T*)p.out + to * p.H + at;
            if constexpr (VEC) *reinterpret_cast<piece*>(y) = r < 0 ? zero : v;
            else *y = r < 0 ? zero[0] : v[0];
        }
    }
}

// out[token] = the sum over its slots of weight * x[place]
template <typename T, bool VEC>
__global__ void __launch_bounds__(kRouteLanes) moe_unpermute_kernel(const MoeRouteParams p) {
    const int64_t token = blockIdx.x, places = p.tokens * p.top_k;
    const int* rows = p.rows + token * p.top_k;
    const int lanes = (int)blockDim.x;
    for (int at = ((int)blockIdx.y * lanes + (int)threadIdx.x) * 8; at < p.H; at += (int)gridDim.y * lanes * 8) {
        v8f_q sum;
#pragma unroll
        for (int k = 0; k < 8; ++k) sum[k] = 0.f;
        for (int j = 0; j < p.top_k; ++j) {
            const int64_t r = rows[j];
            if (r < 0 || r >= places) continue;
            const v8f_q v = get8<T, VEC>((const T*)p.x + r * p.H, at, p.H);
            const float w = weight_of(p.weights, p.weights_type, token * p.top_k + j);
#pragma unroll
            for (int k = 0; k < 8; ++k) sum[k] = __builtin_fmaf(w, v[k], sum[k]);
        }
        set8<T, VEC>((T*)p.out + token * p.H, at, p.H, sum);
    }
}

// out[place] = weight * x[token]; grad_weights[slot] = <x[token], made[place]>
template <typename T, bool VEC>
__global__ void __launch_bounds__(kRouteLanes) moe_unpermute_backward_kernel(const MoeRouteParams p) {
    __shared__ float part[kRouteLanes / 64];
    const int64_t token = blockIdx.x, places = p.tokens * p.top_k;
    const int tid = threadIdx.x, lanes = (int)blockDim.x;
    const T* x = (const T*)p.x + token * p.H;
    const int* rows = p.rows + token * p.top_k;
    for (int j = (int)blockIdx.y; j < p.top_k; j += (int)gridDim.y) {
        const int r = rows[j];
        const int64_t to = r < 0 ? -1 - (int64_t)r : r;
        const bool here = r >= 0 && to < places;
        const float w = weight_of(p.weights, p.weights_type, token * p.top_k + j);
        float dot = 0.f;
        if (to < places) {
            for (int at = tid * 8; at < p.H; at += lanes * 8) {
                v8f_q g = get8<T, VEC>(x, at, p.H);
                if (here) {
                    const v8f_q m = get8<T, VEC>((const T*)p.made + to * p.H, at, p.H);
#pragma unroll
                    for (int k = 0; k < 8; ++k) dot = __builtin_fmaf(g[k], m[k], dot);
                    g *= w;
                } else {
                    g = 0.f;
                }
                set8<T, VEC>((T*)p.out + to * p.H, at, p.H, g);
            }
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) dot += __shfl_xor(dot, d);
        if (tid % 64 == 0) part[tid / 64] = dot;
        __syncthreads();
        if (tid == 0) {
            float sum = 0.f;
            for (int i = 0; i < lanes / 64; ++i) sum += part[i];
            const int64_t at = token * p.top_k + j;
            if (p.weights_type == OUT_F32) ((float*)p.grad_weights)[at] = sum;
            else if (p.weights_type == OUT_BF16) ((__bf16*)p.grad_weights)[at] = (__bf16)sum;
            else ((_Float16*)p.grad_weights)[at] = (_Float16)sum;
        }
        __syncthreads();
    }
}

template <typename T, bool VEC>
hipError_t launch(int which, const MoeRouteParams& p, hipStream_t s) {
    // A lane per piece of a row, up to kRouteLanes (16384 x 6 of 1024 bf16 with 128 lanes instead of 256: the gradient 120 -> 106 us), and workgroups that
    // share a longer row (3001 x 8 of 4096 fp32: permute, with pieces of 16 bytes instead of 32, 113 -> 93 us).
    const int piece = which != 0 ? 8 : VEC ? 16 / sizeof(T) : 1;
    const int64_t pieces = ((int64_t)p.H + piece - 1) / piece;
    const int lanes = pieces <= 64 ? 64 : pieces <= 128 ? 128 : kRouteLanes;
    // The gradient of few pairs: a workgroup per pair instead of per token (bf16 rows of 2048, 6 per token, us: 16 tokens 9.7 -> 6.6, 300 12.6 -> 7.5, 1000 15.3 -> 13.2;
    // 2000 24.8 -> 26.7, 4096 45 -> 51).
    int64_t parts = which != 2 ? (pieces + lanes - 1) / lanes : p.tokens * p.top_k <= kRoutePairs ? p.top_k : 1;
    if (parts == 0) return hipSuccess;  // rows of no elements, or none
    if (parts * p.tokens > kRouteParts) parts = kRouteParts / p.tokens > 0 ? kRouteParts / p.tokens : 1;
    const dim3 grid((unsigned)p.tokens, (unsigned)parts), block(lanes);
    if (which == 0) hipLaunchKernelGGL((moe_permute_kernel<T, VEC>), grid, block, 0, s, p);
    else if (which == 1) hipLaunchKernelGGL((moe_unpermute_kernel<T, VEC>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((moe_unpermute_backward_kernel<T, VEC>), grid, block, 0, s, p);
    return hipGetLastError();
}
hipError_t launch_type(int which, const MoeRouteParams& p, int type, hipStream_t s) {
    if (p.tokens <= 0) return hipSuccess;
    if (type == OUT_F32) return p.vec ? launch<float, true>(which, p, s) : launch<float, false>(which, p, s);
    if (type == OUT_BF16) return p.vec ? launch<__bf16, true>(which, p, s) : launch<__bf16, false>(which, p, s);
    if (type == OUT_F16) return p.vec ? launch<_Float16, true>(which, p, s) : launch<_Float16, false>(which, p, s);
    return hipErrorInvalidValue;
}

}  // namespace

namespace {
// Pairs that are sorted in one launch (64 experts, int64, us, one launch / two): 4096 4.9 / 6.8, 16384 6.7 / 7.2, 24576 7.9 / 7.4, 262144 43 / 12; 8 experts
// 16384 7.9 / 6.9, 256 experts 24576 8.3 / 9.4.
constexpr int64_t kSortAlone = 16384;
constexpr int kSortGroups = 256;
// A wave's slice is a multiple of 64 pairs, a workgroup's at least 1024.
struct SortPlan { int groups, per_wave; };
SortPlan sort_plan(int64_t n) {
    int64_t groups = (n + 64 * kSortWaves - 1) / (64 * kSortWaves);
    groups = groups < 1 ? 1 : groups > kSortGroups ? kSortGroups : groups;
    const int64_t waves = groups * kSortWaves, per_wave = ((n + waves - 1) / waves + 63) / 64 * 64;
    return {(int)groups, per_wave > 0 ? (int)per_wave : 64};
}
template <typename IdT>
hipError_t launch_sort(const IdT* ids, int n, int E, int* counts, int* indptr, int* rows, int* slots, hipStream_t s) {
    const SortPlan plan = sort_plan(n);
    const dim3 grid(plan.groups), block(64 * kSortWaves);
    const int bytes = ((kSortWaves + 2) * (E + 1) + kSortWaves) * 4;
    if (n <= kSortAlone) {
        hipLaunchKernelGGL((moe_sort_kernel<IdT, false>), grid, block, bytes, s, ids, n, E, plan.per_wave, nullptr, indptr, rows, slots);
        return hipGetLastError();
    }
    hipLaunchKernelGGL((moe_count_kernel<IdT>), grid, block, (E + 1) * 4, s, ids, n, E, plan.per_wave, counts);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((moe_sort_kernel<IdT, true>), grid, block, bytes, s, ids, n, E, plan.per_wave, counts, indptr, rows, slots);
    return hipGetLastError();
}
}  // namespace

int64_t moe_sort_workspace_bytes(int64_t n, int E) { return n <= kSortAlone ? 0 : (int64_t)sort_plan(n).groups * (E + 1) * 4; }

hipError_t run_moe_sort(const void* ids, bool ids_are_i64, int n, int E, int* counts, int* indptr, int* rows, int* slots, hipStream_t s) {
    if (E < 1 || E > kSortMaxExperts) return hipErrorInvalidValue;
    return ids_are_i64 ? launch_sort((const int64_t*)ids, n, E, counts, indptr, rows, slots, s) : launch_sort((const int*)ids, n, E, counts, indptr, rows, slots, s);
}

int64_t moe_route_threads(const MoeRouteParams& p) { return p.tokens * kRouteLanes; }
hipError_t run_moe_permute(const MoeRouteParams& p, int type, hipStream_t s) { return launch_type(0, p, type, s); }
hipError_t run_moe_unpermute(const MoeRouteParams& p, int type, hipStream_t s) { return launch_type(1, p, type, s); }
hipError_t run_moe_unpermute_backward(const MoeRouteParams& p, int type, hipStream_t s) { return launch_type(2, p, type, s); }

}  // namespace tg
