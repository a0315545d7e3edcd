// The entry point of the tokens drawn from given random numbers (draw.cuh); see include/rsv_b200.h for the contract.
#include "draw_cluster.cuh"

#include <algorithm>

#include "entry.hpp"
#include "rsv_b200.h"

namespace rsv {

// V weights of up to 2^F fit 62 bits, and the up to 384 of a thread 53: those are summed in fp64
static int draw_bits(int64_t V) {
    int lg = 0;
    while ((int64_t(1) << lg) < V) ++lg;
    return lg > 16 ? 62 - lg : 46;  // (384 a thread: V from 2^19 on, F = 43)
}

template <typename T>
static void launch_draw(cudaStream_t stream, int device, int64_t rows, const DrawArgs& A) {
    constexpr int N = DcVec<T>::n, unit = kDwThreads * N, most = kDcSliceBytes / (int)sizeof(T);  // a warp's stretch is whole vectors for all lanes
    const bool aligned = reinterpret_cast<uintptr_t>(A.logits) % 16 == 0 && (rows == 1 || A.ld * sizeof(T) % 16 == 0);
    const int64_t places = (int64_t)A.V + (aligned ? 0 : N - 1);
    int S = 1;
    while (S < kDcMaxCtas && (int64_t)S * most < places) S *= 2;
    if ((int64_t)S * (kDcMostSliceBytes / (int64_t)sizeof(T)) < places + S * unit) {
        draw_plain_kernel<T><<<(unsigned)rows, kDwThreads, 0, stream>>>(A);
        RSV_CUDA(cudaGetLastError());
        return;
    }
    // Few rows: over more CTAs, as long as two for each SM suffice.  One row of 16384 logits: 9.3 us with eight CTAs (top-k 50), 10.9 with as many as its size asks for; 74 rows of
    // 32000: 14.1 with eight, 12.4 with four.
    while (S < kDcMaxCtas && rows * S * 2 <= 2 * 148 && places > (int64_t)S * 4 * unit) S *= 2;
    const int slice = (int)((places + (int64_t)S * unit - 1) / ((int64_t)S * unit)) * unit;
    const size_t smem = sizeof(DcShared) + std::max((size_t)slice * sizeof(T), sizeof(DwPlainShared));
    static bool configured[64] = {false};
    if (device >= 64 || !configured[device]) {
        RSV_CUDA(cudaFuncSetAttribute(draw_cluster_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(sizeof(DcShared) + kDcMostSliceBytes)));
        if (device < 64) configured[device] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * S));
    cfg.blockDim = dim3(kDwThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute at[1] = {};
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)S;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    RSV_CUDA(cudaLaunchKernelEx(&cfg, draw_cluster_kernel<T>, A, S, slice));
}

void engine_draw(cudaStream_t stream, int device, int dtype, const void* logits_dev, int64_t rows, int64_t V, int64_t row_stride, const float* params4_dev,
                 const float* uniforms_dev, uint32_t* tokens_dev, float* logprobs_dev) {
    DrawArgs A = {logits_dev, row_stride, (int)V, draw_bits(V), params4_dev, uniforms_dev, tokens_dev, logprobs_dev};
    if (dtype == RSV_F32)
        launch_draw<float>(stream, device, rows, A);
    else if (dtype == RSV_F16)
        launch_draw<__half>(stream, device, rows, A);
    else
        launch_draw<__nv_bfloat16>(stream, device, rows, A);
}

}  // namespace rsv

extern "C" int rsv_draw_tokens(int device, void* stream, int dtype, const void* logits_dev, int64_t rows, int64_t V, int64_t row_stride, const float* params4_dev,
                               const float* uniforms_dev, uint32_t* tokens_dev, float* logprobs_dev) {
    using namespace rsv;
    return entry_guarded([&] {
        if (rows < 0) throw std::runtime_error("draw_tokens: negative number of rows");
        if (dtype != RSV_F32 && dtype != RSV_F16 && dtype != RSV_BF16) throw std::runtime_error("draw_tokens: dtype must be RSV_F32, RSV_F16 or RSV_BF16");
        if (V < 1 || V > (int64_t(1) << kDwMaxLogV)) throw std::runtime_error("draw_tokens: V must be between 1 and 2^22");
        if (rows > 0x7fffffffLL / 8) throw std::runtime_error("draw_tokens: too many rows");
        if (row_stride < 0) throw std::runtime_error("draw_tokens: negative row stride");
        if (rows == 0) return;
        if (!logits_dev || !params4_dev || !uniforms_dev || !tokens_dev) throw std::runtime_error("draw_tokens: null argument");
        const uintptr_t size = dtype == RSV_F32 ? 4 : 2;
        if ((uintptr_t)logits_dev % size || (uintptr_t)params4_dev % 4 || (uintptr_t)uniforms_dev % 4 || (uintptr_t)tokens_dev % 4 || (uintptr_t)logprobs_dev % 4)
            throw std::runtime_error("draw_tokens: a pointer is not aligned to its type");
        DeviceScope on(device);
        engine_draw((cudaStream_t)stream, device, dtype, logits_dev, rows, V, row_stride, params4_dev, uniforms_dev, tokens_dev, logprobs_dev);
    });
}
