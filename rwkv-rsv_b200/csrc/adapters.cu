// The entry point of the low-rank adapters (adapters.cuh); see include/rsv_b200.h for the contract.
#include "adapters.cuh"

#include "entry.hpp"
#include "rsv_b200.h"

namespace rsv {

template <typename X, typename W>
static void launch_adapters(cudaStream_t stream, const AdapterArgs& P) {
    adapters_row_kernel<X, W><<<(unsigned)P.rows, kAdThreads, 0, stream>>>(P);
    RSV_CUDA(cudaGetLastError());
}

void engine_adapters(cudaStream_t stream, int xtype, int wtype, const AdapterArgs& P) {
    if (xtype == RSV_F16)
        launch_adapters<__half, __half>(stream, P);
    else if (xtype == RSV_BF16)
        launch_adapters<__nv_bfloat16, __nv_bfloat16>(stream, P);
    else if (wtype == RSV_F16)
        launch_adapters<float, __half>(stream, P);
    else
        launch_adapters<float, __nv_bfloat16>(stream, P);
}

// First and one past the last byte of `rows` rows of `cols` elements.
static void span(const void* p, int64_t rows, int64_t cols, int64_t ld, int64_t size, uintptr_t& lo, uintptr_t& hi) {
    lo = (uintptr_t)p;
    hi = lo + (uintptr_t)(((rows - 1) * ld + cols) * size);
}

}  // namespace rsv

extern "C" int rsv_adapters_apply(int device, void* stream, const rsv_adapters* ad, int xtype, const void* x_dev, int64_t x_stride, int64_t rows,
                                  const int32_t* index_dev, const void* base_dev, int64_t base_stride, void* out_dev, int64_t out_stride) {
    using namespace rsv;
    return entry_guarded([&] {
        if (!ad) throw std::runtime_error("adapters: null argument");
        if (ad->dtype != RSV_F16 && ad->dtype != RSV_BF16) throw std::runtime_error("adapters: the adapters' dtype must be RSV_F16 or RSV_BF16");
        if (xtype != RSV_F32 && xtype != ad->dtype) throw std::runtime_error("adapters: activations must be RSV_F32 or of the adapters' dtype");
        const int64_t lim = 0x7fffffffLL;
        if (ad->K < 1 || ad->M < 1 || ad->slots < 1 || ad->K > lim / 8 || ad->M > lim / 8 || ad->slots > 65536)
            throw std::runtime_error("adapters: K and M must be between 1 and 2^28 - 1, slots between 1 and 65536");
        if (ad->max_rank < 1 || ad->max_rank > kAdMaxRank) throw std::runtime_error("adapters: max_rank must be between 1 and 256");
        if (ad->a_row < 0 || ad->a_slot < 0 || ad->b_row < 0 || ad->b_slot < 0 || x_stride < 0 || base_stride < 0) throw std::runtime_error("adapters: negative stride");
        if (rows < 0 || rows > lim / 64) throw std::runtime_error("adapters: rows must be between 0 and 2^25");
        if (rows == 0) return;
        if (!ad->a || !ad->b || !x_dev || !index_dev || !out_dev) throw std::runtime_error("adapters: null argument");
        if (rows > 1 && out_stride < ad->M) throw std::runtime_error("adapters: rows of out overlap");
        const int64_t xs = xtype == RSV_F32 ? 4 : 2;
        if ((uintptr_t)x_dev % xs || (uintptr_t)base_dev % xs || (uintptr_t)out_dev % xs || (uintptr_t)ad->a % 2 || (uintptr_t)ad->b % 2 || (uintptr_t)index_dev % 4 ||
            (uintptr_t)ad->ranks % 4 || (uintptr_t)ad->scales % 4)
            throw std::runtime_error("adapters: a pointer is not aligned to its type");
        uintptr_t o0, o1, p0, p1;
        span(out_dev, rows, ad->M, out_stride, xs, o0, o1);
        span(x_dev, rows, ad->K, x_stride, xs, p0, p1);
        if (o0 < p1 && p0 < o1) throw std::runtime_error("adapters: out and x overlap");
        if (base_dev && !(base_dev == out_dev && (base_stride == out_stride || rows == 1))) {
            span(base_dev, rows, ad->M, base_stride, xs, p0, p1);
            if (o0 < p1 && p0 < o1) throw std::runtime_error("adapters: out and base overlap without being the same rows");
        }
        DeviceScope on(device);
        AdapterArgs P = {x_dev, index_dev, ad->a, ad->b, ad->ranks, ad->scales, base_dev, out_dev, x_stride, base_stride, out_stride, ad->a_slot, ad->a_row, ad->b_slot, ad->b_row,
                         (int)rows, (int)ad->K, (int)ad->M, (int)ad->slots, (int)ad->max_rank};
        engine_adapters((cudaStream_t)stream, xtype, ad->dtype, P);
    });
}
