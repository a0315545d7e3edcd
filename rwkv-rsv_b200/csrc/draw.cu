// The entry point of the tokens drawn from given random numbers (draw.cuh); see include/rsv_b200.h for the contract.
#include "draw.cuh"

#include "entry.hpp"
#include "rsv_b200.h"

namespace rsv {

// rint(2^F) V fits 63 bits, and a weight 51
static int draw_bits(int64_t V) {
    int lg = 0;
    while ((int64_t(1) << lg) < V) ++lg;
    return lg > 12 ? 62 - lg : 50;
}

void engine_draw(cudaStream_t stream, int dtype, const void* logits_dev, int64_t rows, int64_t V, int64_t row_stride, const float* params4_dev,
                 const float* uniforms_dev, uint32_t* tokens_dev, float* logprobs_dev) {
    DrawArgs A = {logits_dev, row_stride, (int)V, draw_bits(V), params4_dev, uniforms_dev, tokens_dev, logprobs_dev};
    if (dtype == RSV_F32)
        draw_plain_kernel<float><<<(unsigned)rows, kDwThreads, 0, stream>>>(A);
    else if (dtype == RSV_F16)
        draw_plain_kernel<__half><<<(unsigned)rows, kDwThreads, 0, stream>>>(A);
    else
        draw_plain_kernel<__nv_bfloat16><<<(unsigned)rows, kDwThreads, 0, stream>>>(A);
    RSV_CUDA(cudaGetLastError());
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
        engine_draw((cudaStream_t)stream, dtype, logits_dev, rows, V, row_stride, params4_dev, uniforms_dev, tokens_dev, logprobs_dev);
    });
}
