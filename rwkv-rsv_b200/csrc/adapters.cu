// The entry point of the low-rank adapters (adapters.cuh); see include/rsv_b200.h for the contract.
#include "adapters.cuh"

#include <algorithm>
#include <initializer_list>

#include "entry.hpp"
#include "rsv_b200.h"

namespace rsv {

// Tiles of a block of rows if they are shared evenly among the adapters: about one in two adapters has a tile that is not full.
static int64_t expected_tiles(const AdapterArgs& P, int T) {
    const int rows = std::min(P.rows, kAdBlockRows), adapters = std::min(P.slots, rows);
    return std::max(adapters, rows / T + adapters / 2);
}

template <typename X, typename W, int MT, int STAGES>
static void launch_tiles(cudaStream_t stream, int device, AdapterArgs P) {
    typedef AdShape<X, W, MT, STAGES> Z;
    constexpr int T = Z::T;
    P.block_rows = std::min(P.rows, kAdBlockRows);
    const int blocks = (P.rows + P.block_rows - 1) / P.block_rows;
    P.tiles = std::min(P.block_rows, P.block_rows / T + std::min(P.slots + P.copies, P.block_rows));
    // Two CTAs fit on an SM, and one round of them is the fastest: 64 sessions of 10240 k on 64 adapters take 20 us as 256 CTAs (25 with three on an SM, whose
    // registers spill).  Any number of CTAs is a cluster: 50 such sessions take 17.2 us with five CTAs each and 19.0 with four.  (The tiles that will be there,
    // not those that may be.)
    P.S = kAdMaxCtas;
    while (P.S > 1 && blocks * expected_tiles(P, T) * P.S > 2 * 148) --P.S;
    const size_t smem = Z::smem(P.rank_cap);
    static bool configured[64] = {false};
    if (device >= 64 || !configured[device]) {
        RSV_CUDA(cudaFuncSetAttribute(adapters_kernel<X, W, MT, STAGES>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Z::smem(Z::most_rank)));
        if (device < 64) configured[device] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((int64_t)blocks * P.tiles * P.S));
    cfg.blockDim = dim3(kAdThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute at[1] = {};
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)P.S;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    RSV_CUDA(cudaLaunchKernelEx(&cfg, adapters_kernel<X, W, MT, STAGES>, P));
}

template <typename X, typename W>
static void launch_adapters(cudaStream_t stream, int device, AdapterArgs P) {
    const int rows = std::min(P.rows, kAdBlockRows), each = rows / std::min(P.slots, rows);  // rows of an adapter, if they are shared evenly
    // Larger tiles read the adapters less often, but leave fewer CTAs side by side and split x more often: where sixteen rows' activations are under two thirds of
    // an adapter, and enough tiles are left for the GPU.  us with tiles of 16, 32 and 64 rows, by that proportion: bf16, 4096 rows, 64 ranks, 2560 x 10240 (0.45)
    // 100, 87, 76; 2048 rows, 256 ranks, 2560 x 2560 (0.1) 84, 76; 128 ranks (0.2) 49, 44, 96 (one CTA per SM: so 64 rows for up to 64 ranks); fp32, 4096 rows, 64
    // ranks (0.75) 56, 53, 57; 1024 rows, 32 ranks (1.5) 17.3, 18.7; 4096 rows, 16 ranks (3) 37, 55, 51.  Fewer tiles than the 240 CTAs: 1024 rows, 32 ranks in
    // tiles of 64 rows 26.5.
    const int64_t xs = sizeof(X), adapter = (int64_t)P.rank_cap * (P.K + P.M) * 2, sixteen = 16 * xs * (P.K + (int64_t)P.M * (P.base ? 2 : 1));
    const auto fits = [&](int T) { return 2 * adapter >= 3 * sixteen && each >= T * 3 / 4 && expected_tiles(P, T) * kAdMaxCtas >= 240; };
    if (P.rank_cap <= kAdChunk && fits(64))
        launch_tiles<X, W, 4, sizeof(X) == 4 ? 2 : 3>(stream, device, P);
    else if (fits(32))
        launch_tiles<X, W, 2, 3>(stream, device, P);
    // five stages where they fit twice on an SM: 64 sessions of 10240 k 19.9 us, with three 20.7
    else if (P.rank_cap <= 32)
        launch_tiles<X, W, 1, 5>(stream, device, P);
    else
        launch_tiles<X, W, 1, 3>(stream, device, P);
}

void engine_apply_adapters(cudaStream_t stream, int device, const rsv_adapters& ad, int xtype, const void* x, int64_t x_stride, int64_t rows, const int32_t* index,
                           const void* base, int64_t base_stride, void* out, int64_t out_stride) {
    AdapterArgs P = {x, index, ad.a, ad.b, ad.ranks, ad.scales, base, out, x_stride, base_stride, out_stride, ad.a_slot, ad.a_row, ad.b_slot, ad.b_row, (int)rows, (int)ad.K, (int)ad.M,
                     (int)ad.slots, (int)ad.max_rank};
    const int wtype = ad.dtype;
    const int xs = xtype == RSV_F32 ? 4 : 2;
    const auto at = [](int bytes, const void* p, int64_t size, std::initializer_list<int64_t> strides) {  // rows start at multiples of `bytes`
        bool ok = (uintptr_t)p % bytes == 0;
        for (int64_t s : strides) ok = ok && s * size % bytes == 0;
        return ok ? 1 : 0;
    };
    P.wide_x = at(16, P.x, xs, {P.ldx});
    P.wide_a = at(16, P.a, 2, {P.a_slot, P.a_row});
    P.wide_b = at(16, P.b, 2, {P.b_slot, P.b_row});
    P.wide_base = at(16, P.base, xs, {P.ldbase});
    P.wide_out = at(4 * xs, P.out, xs, {P.ldout});
    P.copies = P.base != P.out;
    P.rank_cap = (P.max_rank + 15) / 16 * 16;
    if (xtype == RSV_F16)
        launch_adapters<__half, __half>(stream, device, P);
    else if (xtype == RSV_BF16)
        launch_adapters<__nv_bfloat16, __nv_bfloat16>(stream, device, P);
    else if (wtype == RSV_F16)
        launch_adapters<float, __half>(stream, device, P);
    else
        launch_adapters<float, __nv_bfloat16>(stream, device, P);
}

// Rows of `cols` elements, ld elements apart.
struct Span {
    const void* p;
    int64_t cols, ld;
};
// Whether an element of a's rows may be one of b's: by the first and last bytes, and, for rows the same distance apart, by columns (x and out may be columns of one array).
static bool meet(const Span& a, const Span& b, int64_t rows, int64_t size) {
    const uintptr_t a0 = (uintptr_t)a.p, a1 = a0 + (uintptr_t)(((rows - 1) * a.ld + a.cols) * size), b0 = (uintptr_t)b.p, b1 = b0 + (uintptr_t)(((rows - 1) * b.ld + b.cols) * size);
    if (a1 <= b0 || b1 <= a0) return false;
    if (a.ld != b.ld || a.ld == 0) return true;
    const int64_t pitch = a.ld * size;
    int64_t at = (int64_t)(b0 - a0) % pitch;  // where a row of b begins behind one of a
    if (at < 0) at += pitch;
    return at < a.cols * size || at + b.cols * size > pitch;
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
        if (ad->K < 1 || ad->M < 1 || ad->slots < 1 || ad->K > lim / 8 || ad->M > lim / 8 || ad->slots > kAdMaxSlots)
            throw std::runtime_error("adapters: K and M must be between 1 and 2^28 - 1, slots between 1 and 4096");
        if (ad->max_rank < 1 || ad->max_rank > kAdMaxRank) throw std::runtime_error("adapters: max_rank must be between 1 and 256");
        if (ad->a_row < 0 || ad->a_slot < 0 || ad->b_row < 0 || ad->b_slot < 0 || x_stride < 0 || base_stride < 0) throw std::runtime_error("adapters: negative stride");
        if (rows < 0 || rows > kAdMaxRows) throw std::runtime_error("adapters: rows must be between 0 and " + std::to_string(kAdMaxRows));
        if (rows == 0) return;
        if (!ad->a || !ad->b || !x_dev || !index_dev || !out_dev) throw std::runtime_error("adapters: null argument");
        if (rows > 1 && out_stride < ad->M) throw std::runtime_error("adapters: rows of out overlap");
        const int64_t xs = xtype == RSV_F32 ? 4 : 2;
        if ((uintptr_t)x_dev % xs || (uintptr_t)base_dev % xs || (uintptr_t)out_dev % xs || (uintptr_t)ad->a % 2 || (uintptr_t)ad->b % 2 || (uintptr_t)index_dev % 4 ||
            (uintptr_t)ad->ranks % 4 || (uintptr_t)ad->scales % 4)
            throw std::runtime_error("adapters: a pointer is not aligned to its type");
        const Span out = {out_dev, ad->M, out_stride};
        if (meet(out, {x_dev, ad->K, x_stride}, rows, xs)) throw std::runtime_error("adapters: out and x overlap");
        if (base_dev && !(base_dev == out_dev && (base_stride == out_stride || rows == 1)) && meet(out, {base_dev, ad->M, base_stride}, rows, xs))
            throw std::runtime_error("adapters: out and base overlap without being the same rows");
        DeviceScope on(device);
        engine_apply_adapters((cudaStream_t)stream, device, *ad, xtype, x_dev, x_stride, rows, index_dev, base_dev, base_stride, out_dev, out_stride);
    });
}
