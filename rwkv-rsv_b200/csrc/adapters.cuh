// Low-rank adapters of many requests at once, beside a projection that all rows share:
//   out[n] = base[n] + scale[a] B[a] (A[a] x[n]),  a = index[n]; rows with an index outside 0 .. slots - 1 have no adapter: out[n] = base[n].
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace rsv {

struct AdapterArgs {
    const void* x;
    const int32_t* index;
    const void *a, *b;  // [slots][max_rank][K], [slots][M][max_rank]
    const int32_t* ranks;  // may be null: max_rank
    const float* scales;   // may be null: 1
    const void* base;      // may be null: 0
    void* out;
    int64_t ldx, ldbase, ldout, a_slot, a_row, b_slot, b_row;
    int rows, K, M, slots, max_rank;
};

__device__ __forceinline__ float ad_f32(float v) { return v; }
__device__ __forceinline__ float ad_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float ad_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename X>
__device__ __forceinline__ X ad_round(float v);
template <>
__device__ __forceinline__ float ad_round<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half ad_round<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 ad_round<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

constexpr int kAdThreads = 256;
constexpr int kAdMaxRank = 256;

// A row by one CTA: a warp per row of A, a thread per output.
template <typename X, typename W>
__global__ void __launch_bounds__(kAdThreads) adapters_row_kernel(AdapterArgs P) {
    __shared__ float t[kAdMaxRank];
    const int n = blockIdx.x, tid = threadIdx.x;
    const X* x = reinterpret_cast<const X*>(P.x) + (int64_t)n * P.ldx;
    const X* base = P.base ? reinterpret_cast<const X*>(P.base) + (int64_t)n * P.ldbase : nullptr;
    X* out = reinterpret_cast<X*>(P.out) + (int64_t)n * P.ldout;
    const int a = P.index[n];
    const bool has = a >= 0 && a < P.slots;
    const int rank = has ? (P.ranks ? max(0, min(P.ranks[a], P.max_rank)) : P.max_rank) : 0;
    const float scale = has && P.scales ? P.scales[a] : 1.f;
    for (int r = tid >> 5; r < rank; r += kAdThreads / 32) {
        const W* w = reinterpret_cast<const W*>(P.a) + a * P.a_slot + r * P.a_row;
        float s = 0.f;
        for (int k = tid & 31; k < P.K; k += 32) s = fmaf(ad_f32(x[k]), ad_f32(w[k]), s);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if ((tid & 31) == 0) t[r] = s;
    }
    __syncthreads();
    for (int m = tid; m < P.M; m += kAdThreads) {
        const W* w = reinterpret_cast<const W*>(P.b) + (has ? a * P.b_slot + m * P.b_row : 0);
        float s = 0.f;
        for (int r = 0; r < rank; ++r) s = fmaf(t[r], ad_f32(w[r]), s);
        const float y = base ? ad_f32(base[m]) : 0.f;
        out[m] = ad_round<X>(rank ? fmaf(scale, s, y) : y);
    }
}

}  // namespace rsv
