// One token per row of logits from a given random number u, after temperature T, top-k, top-p and min-p.
//
// With y_i = (l_i - max) log2(e) / T and w_i = 2^y_i (0 where y_i < -40):
//   top-k   the k largest logits are kept, equal ones by their index;
//   top-p   of these, in falling order, those before which the sum of w is under p times the sum over all that top-k kept;
//   min-p   of these, the ones with w > 0 and w >= min_p;
//   draw    the first kept token, in vocabulary order, whose running sum of w exceeds u times the sum of all kept.
// So the kept tokens are the ones down to a cut: a logit and, among the logits equal to it, a number of lowest indices.
//
// The weights are whole numbers: rint(w 2^F) in 64 bits, with F such that V of them fit.  y and w are computed in fp64 (fp32 cannot tell the
// running sums of neighbouring tokens apart: of 65536 equal logits each is 1.5e-5 of the sum, and fp32 leaves errors of 1e-7: one row in a hundred
// would draw its neighbour).  Sums of whole numbers do not depend on their order, so neither do the tokens on how a row is split over threads and
// CTAs, and no atomic addition changes a result.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace rsv {

constexpr int kDwThreads = 256;
constexpr int kDwWarps = kDwThreads / 32;
constexpr int kDwMaxLogV = 22;
constexpr uint32_t kDwNone = 0xFFFFFFFFu;  // the token of a row that has none

typedef unsigned long long u64;

struct DrawArgs {
    const void* logits;
    int64_t ld;
    int V, F;
    const float* params4;  // [rows][4]: temperature, bits of top_k, top_p, min_p
    const float* u;
    uint32_t* tokens;
    float* logprobs;  // may be null
};

__device__ __forceinline__ float dw_f32(float v) { return v; }
__device__ __forceinline__ float dw_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float dw_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
// Bits that are ordered like the values; -0 counts as 0.
__device__ __forceinline__ uint32_t dw_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float dw_value(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key); }

// What a row asks for, and its largest logit once that is known.
struct DwRow {
    double c, ymin, mxd;  // log2(e) / T; the least y that min-p keeps
    float T, mx, top_p, min_p;
    uint32_t top_k;  // 0: all
    int F;
    bool greedy;
};
__device__ __forceinline__ DwRow dw_asked(const DrawArgs& A, int row) {
    const float* p = A.params4 + (size_t)row * 4;
    const uint32_t k = __float_as_uint(p[1]);
    DwRow r;
    r.T = p[0];
    r.greedy = !(r.T > 0.f);
    r.top_k = k < (uint32_t)A.V ? k : 0u;
    r.top_p = p[2] > 0.f && p[2] < 1.f ? p[2] : 0.f;
    r.min_p = p[3] > 0.f ? fminf(p[3], 1.f) : 0.f;
    r.F = A.F;
    r.c = r.ymin = r.mxd = 0.0;
    r.mx = 0.f;
    return r;
}
__device__ __forceinline__ double dw_rate(float T) { return 1.4426950408889634074 / (double)T; }
__device__ __forceinline__ double dw_least(float min_p) { return min_p > 0.f ? fmax(log2((double)min_p), -40.0) : -40.0; }
// (The difference first: at a low temperature max and l alone would be too large to subtract.)
__device__ __forceinline__ double dw_y(const DwRow& r, float l) { return ((double)l - r.mxd) * r.c; }

// rint(2^(y + F)) for y = (l - max) c from -40 to 0.  2^y = 2^n 2^(j/16) 2^f with |f| <= 1/32: a table of 2^(F + j/16) and the Taylor polynomial of
// e^(f ln 2) to the fifth power, with the powers of ln 2 in its coefficients (the next term is under 1.5e-13 of the weight).  Kernels that sum weights
// are bound by these eleven fp64 operations and their surroundings (64 of them a cycle and SM).
__device__ __forceinline__ double dw_whole(const DwRow& r, float l, const double* tab16) {
    const double big = 6755399441055744.0 / 16.0, round = 4503599627370496.0, d = (double)l - r.mxd;  // 1.5 2^48: a sum's last place is 1/16; 2^52: it is 1
    const double t = fma(d, r.c, big), f = fma(d, r.c, -(t - big));
    const int n16 = __double2loint(t);
    double p = fma(f, 0.0013333558146428443, 0.0096181291076284769);
    p = fma(p, f, 0.055504108664821583);
    p = fma(p, f, 0.24022650695910072);
    p = fma(p, f, 0.69314718055994529);
    p = fma(p, f, 1.0);
    const double w = tab16[n16 & 15];
    return fma(p, __hiloint2double(__double2hiint(w) + (n16 & ~15) * 65536, __double2loint(w)), round) - round;
}
__device__ __forceinline__ u64 dw_fixed(const DwRow& r, float l, const double* tab16) { return (u64)dw_whole(r, l, tab16); }
// The weight of a logit; 0 for y < -40.
__device__ __forceinline__ u64 dw_weight(const DwRow& r, float l, const double* tab16) { return dw_y(r, l) >= -40.0 ? dw_fixed(r, l, tab16) : 0ull; }
// 2^(j/16)
__constant__ double kDwTable[16] = {1.0,
                                    1.0442737824274138,
                                    1.0905077326652577,
                                    1.1387886347566916,
                                    1.189207115002721,
                                    1.241857812073484,
                                    1.2968395546510096,
                                    1.3542555469368927,
                                    1.4142135623730951,
                                    1.4768261459394993,
                                    1.5422108254079407,
                                    1.6104903319492543,
                                    1.681792830507429,
                                    1.7562521603732995,
                                    1.8340080864093424,
                                    1.9152065613971474};
__device__ __forceinline__ void dw_fill_table(double* tab16, int F) {
    if (threadIdx.x < 16) {
        const double t = kDwTable[threadIdx.x];
        tab16[threadIdx.x] = __hiloint2double(__double2hiint(t) + (F << 20), __double2loint(t));
    }
}
// top_p of the sum: the sum before a token is under it exactly where it is under the next whole number
__device__ __forceinline__ u64 dw_share(float top_p, u64 total) {
    const u64 P = (u64)ceil((double)top_p * (double)total);
    return P < 1 ? 1 : P > total ? total : P;
}
// u of the sum, so that a running sum exceeds it somewhere
__device__ __forceinline__ u64 dw_target(float u, u64 total) {
    const double x = u > 0.f ? (double)u * (double)total : 0.0;  // (a NaN counts as 0)
    const u64 U = x < (double)total ? (u64)x : total - 1;
    return U < total ? U : total - 1;
}
__device__ __forceinline__ void dw_result(const DrawArgs& A, int row, uint32_t token, float logprob) {
    A.tokens[row] = token;
    if (A.logprobs) A.logprobs[row] = logprob;
}
__device__ __forceinline__ float dw_logprob(const DwRow& r, float l, u64 total) {
    return (float)(dw_y(r, l) * 0.69314718055994530942 - log((double)total * exp2(-(double)r.F)));
}

static_assert(kDwThreads == 256, "a thread per bin of a radix pass");
// ---- a row by one CTA, from global memory -----------------------------------------------------------------
struct DwPlainShared {
    double tab[16];
    u64 hist[256], wsum[kDwWarps], acc;
    uint32_t wcnt[kDwWarps], digit, cnt, best;
    float red[kDwWarps];
};

__device__ __forceinline__ u64 dw_block_sum(u64 v, DwPlainShared& sh) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.wsum[threadIdx.x >> 5] = v;
    __syncthreads();
    u64 t = 0;
#pragma unroll 1
    for (int i = 0; i < kDwWarps; ++i) t += sh.wsum[i];
    return t;
}

// Whole radix passes over the row: slow, but for any input.  (What a row costs here: about 0.3 ms for 65536 logits.)
template <typename T>
__device__ __noinline__ void dw_row_plain(const DrawArgs& A, int row, DwPlainShared& sh) {
    const T* lg = reinterpret_cast<const T*>(A.logits) + (size_t)row * A.ld;
    const int V = A.V, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    DwRow r = dw_asked(A, row);
    r.c = dw_rate(r.T);
    r.ymin = dw_least(r.min_p);
    dw_fill_table(sh.tab, r.F);
    // ---- the largest logit
    float mx = -INFINITY;
    bool nan = false;
    for (int i = tid; i < V; i += kDwThreads) {
        const float l = dw_f32(lg[i]);
        nan |= l != l;
        mx = fmaxf(mx, l);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (lane == 0) sh.red[warp] = mx;
    if (tid == 0) sh.best = kDwNone;
    nan = __syncthreads_or(nan);
    for (int i = 0; i < kDwWarps; ++i) mx = fmaxf(mx, sh.red[i]);
    if (nan || mx == -INFINITY) {
        if (tid == 0) dw_result(A, row, kDwNone, nan ? NAN : -INFINITY);
        return;
    }
    r.mx = mx;
    r.mxd = (double)mx;
    // where there are infinite logits only they are drawn, all alike
    const bool infinite = mx == INFINITY;
    if (infinite) r.mx = 0.f, r.mxd = 0.0;
    const auto logit = [&](int i) {
        const float l = dw_f32(lg[i]);
        return infinite ? (l == INFINITY ? 0.f : -INFINITY) : l;
    };
    if (r.greedy) {
        uint32_t best = kDwNone;
        for (int i = tid; i < V; i += kDwThreads)
            if (logit(i) == r.mx) best = min(best, (uint32_t)i);
        best = __reduce_min_sync(0xffffffffu, best);
        if (lane == 0) atomicMin(&sh.best, best);
        __syncthreads();
        if (tid == 0) dw_result(A, row, sh.best, 0.f);
        return;
    }
    // ---- the cut: logits with a larger key, and the first `equals` of those with this one
    uint32_t cut = 0, equals = 0;
    if (r.top_k) {
        uint32_t prefix = 0, mask = 0, need = r.top_k;
#pragma unroll 1
        for (int shift = 24; shift >= 0; shift -= 8) {
            __syncthreads();
            sh.hist[tid] = 0;
            __syncthreads();
            for (int i = tid; i < V; i += kDwThreads) {
                const uint32_t key = dw_key(logit(i));
                if ((key & mask) == prefix) atomicAdd(reinterpret_cast<uint32_t*>(&sh.hist[(key >> shift) & 255u]), 1u);
            }
            __syncthreads();
            if (tid == 0) {
                uint32_t d = 255, before = 0;
                while (before + (uint32_t)sh.hist[d] < need) before += (uint32_t)sh.hist[d--];
                sh.digit = d;
                sh.cnt = need - before;
            }
            __syncthreads();
            prefix |= sh.digit << shift;
            mask |= 255u << shift;
            need = sh.cnt;
        }
        cut = prefix;
        equals = need;
    }
    if (r.top_p > 0.f) {
        u64 sum = 0;
        for (int i = tid; i < V; i += kDwThreads) {
            const float l = logit(i);
            if (dw_key(l) > cut) sum += dw_weight(r, l, sh.tab);
        }
        const u64 wcut = equals ? dw_weight(r, dw_value(cut), sh.tab) * equals : 0ull;  // the kept ones of those at the cut
        const u64 P = dw_share(r.top_p, dw_block_sum(sum, sh) + wcut);
        uint32_t prefix = 0, mask = 0;
        u64 acc = 0;
#pragma unroll 1
        for (int shift = 24; shift >= 0; shift -= 8) {
            __syncthreads();
            sh.hist[tid] = 0;
            __syncthreads();
            for (int i = tid; i < V; i += kDwThreads) {
                const float l = logit(i);
                const uint32_t key = dw_key(l);
                if ((key & mask) == prefix && key > cut) atomicAdd(&sh.hist[(key >> shift) & 255u], dw_weight(r, l, sh.tab));
            }
            if (tid == 0 && wcut && (cut & mask) == prefix) atomicAdd(&sh.hist[(cut >> shift) & 255u], wcut);
            __syncthreads();
            if (tid == 0) {
                uint32_t d = 255;
                u64 a = acc;
                while (d > 0 && a + sh.hist[d] < P) a += sh.hist[d--];
                sh.digit = d;
                sh.acc = a;
            }
            __syncthreads();
            prefix |= sh.digit << shift;
            mask |= 255u << shift;
            acc = sh.acc;
        }
        const u64 w = dw_weight(r, dw_value(prefix), sh.tab);
        cut = prefix;
        equals = w ? (uint32_t)((P - acc + w - 1) / w) : 1u;
    }
    // ---- the sum of the kept ones
    u64 sum = 0;
    for (int i = tid; i < V; i += kDwThreads) {
        const float l = logit(i);
        const double y = dw_y(r, l);
        if (dw_key(l) > cut && y >= r.ymin) sum += dw_fixed(r, l, sh.tab);
    }
    u64 total = dw_block_sum(sum, sh);
    if (equals && dw_y(r, dw_value(cut)) >= r.ymin) total += dw_weight(r, dw_value(cut), sh.tab) * equals;
    const u64 U = dw_target(A.u[row], total);
    // ---- the draw, 256 tokens at a time in vocabulary order
    u64 run = 0;
    uint32_t seen = 0;
#pragma unroll 1
    for (int i0 = 0; i0 < V; i0 += kDwThreads) {
        const int i = i0 + tid;
        const float l = i < V ? logit(i) : -INFINITY;
        const uint32_t key = dw_key(l);
        const bool eq = i < V && key == cut;
        const uint32_t ballot = __ballot_sync(0xffffffffu, eq);
        __syncthreads();
        if (lane == 0) sh.wcnt[warp] = __popc(ballot);
        __syncthreads();
        uint32_t place = seen + __popc(ballot & ((1u << lane) - 1u));
        for (int j = 0; j < kDwWarps; ++j) {
            if (j < warp) place += sh.wcnt[j];
            seen += sh.wcnt[j];
        }
        const double y = dw_y(r, l);
        u64 w = i < V && y >= r.ymin && (key > cut || (eq && place < equals)) ? dw_fixed(r, l, sh.tab) : 0ull, incl = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 t = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += t;
        }
        if (lane == 31) sh.wsum[warp] = incl;
        __syncthreads();
        u64 base = run;
        for (int j = 0; j < kDwWarps; ++j) {
            if (j < warp) base += sh.wsum[j];
            run += sh.wsum[j];
        }
        if (w && base + incl > U && base + incl - w <= U) dw_result(A, row, (uint32_t)i, dw_logprob(r, l, total));
        if (run > U) break;  // (the same for all threads)
    }
}

template <typename T>
__global__ void __launch_bounds__(kDwThreads) draw_plain_kernel(DrawArgs A) {
    __shared__ DwPlainShared sh;
    dw_row_plain<T>(A, (int)blockIdx.x, sh);
}

}  // namespace rsv
